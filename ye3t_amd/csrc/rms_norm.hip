// Root-mean-square norm of feature rows with the residual's addition, its
// gradient, and its rows in 8 bits.
//
//   h = x + r,   rho = (mean(h^2) + epsilon)^(-1/2),   y = h rho w
//   u = g w,     dh = rho (u - h rho^2 mean(u h)) + gh,   dw = sum over rows of g h rho
//
// Bound by memory: a value is read and written once and takes a dozen
// operations.  A row is held in the registers of a group of L lanes (4, 16 or
// 64 lanes of a wave, or four waves), K chunks of 16 bytes a lane, so that the
// mean and the output come from one read; rows wider than four waves hold are
// read again for the output.  h, the means and the weight's sums are fp32; h
// and y are each rounded once, from the unrounded sum.
#include "rows.h"

namespace ye3t {
namespace {

constexpr int kThreads = 256;
constexpr int kScaleGroup = 128;  // columns that share a scale of the 8-bit rows
constexpr float kLargest8 = 448.0f;

// Sums of two values over the L lanes that share a row; every lane gets the same
// bits.  `part` has two places for each wave.
template <int L>
__device__ inline void row_sums(float& a, float& b, float* part) {
#pragma unroll
  for (int m = 1; m < (L < 64 ? L : 64); m *= 2) {
    const float x = __shfl_xor(a, m), y = __shfl_xor(b, m);
    a += x;
    b += y;
  }
  if constexpr (L > 64) {
    __syncthreads();  // the last sums' parts have been read
    if ((threadIdx.x & 63) == 0) {
      part[2 * (threadIdx.x >> 6)] = a;
      part[2 * (threadIdx.x >> 6) + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) {
      a += part[2 * w];
      b += part[2 * w + 1];
    }
  }
}

// 800 000 x 161 fp32 with the addition: 430 us for 2.06 GB, 4.8 TB/s (a large copy:
// 5.1); to 8 bits, 50 000 x 1 449 fp32: 211 us for 0.94 GB.
enum { kPlain = 0, kEightBit = 1 };

// K: chunks a lane holds; 0: any number, the row is read twice.
template <typename T, int L, int K, int MODE>
__global__ __launch_bounds__(kThreads) void rms_norm_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                            const T* __restrict__ weight, int64_t rows, int W,
                                                            float epsilon, T* __restrict__ total, T* __restrict__ y,
                                                            uint8_t* __restrict__ codes, float* __restrict__ scales) {
  constexpr int V = kChunk<T>;
  constexpr int H = K > 0 ? K : 1;
  __shared__ float part[2 * kThreads / 64];
  const int lane = int(threadIdx.x) % L, per = kThreads / L;
  const int groups = (W + kScaleGroup - 1) / kScaleGroup;
  for (int64_t row = int64_t(blockIdx.x) * per + int(threadIdx.x) / L; row < rows; row += int64_t(gridDim.x) * per) {
    const T* xr = x + row * W;
    const T* rr = residual ? residual + row * W : nullptr;
    T* tr = total ? total + row * W : nullptr;
    float h[H][V];
    auto sum_of = [&](int c, float* out) {
      const Chunk<T, V> a = Chunk<T, V>::load(xr + c, W - c);
#pragma unroll
      for (int q = 0; q < V; ++q) out[q] = float(a.v[q]);
      if (rr) {
        const Chunk<T, V> b = Chunk<T, V>::load(rr + c, W - c);
#pragma unroll
        for (int q = 0; q < V; ++q) out[q] += float(b.v[q]);
      }
    };
    auto keep_total = [&](int c, const float* v) {
      if (!tr) return;
      Chunk<T, V> a;
#pragma unroll
      for (int q = 0; q < V; ++q) a.v[q] = T(v[q]);
      a.store(tr + c, W - c);
    };
    float square = 0.0f;
#pragma unroll
    for (int k = 0, c = lane * V; K > 0 ? k < K : c < W; ++k, c += L * V) {
      float* v = h[K > 0 ? k : 0];
      if (c < W) {
        sum_of(c, v);
      } else {
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = 0.0f;
      }
#pragma unroll
      for (int q = 0; q < V; ++q) square += v[q] * v[q];
    }
    float unused = 0.0f;
    row_sums<L>(square, unused, part);
    const float rho = 1.0f / sqrtf(square / float(W) + epsilon);
#pragma unroll
    for (int k = 0, c = lane * V; K > 0 ? k < K : c < (W + L * V - 1) / (L * V) * (L * V); ++k, c += L * V) {
      float* v = h[K > 0 ? k : 0];
      if (K == 0) {
        if (c < W) {
          sum_of(c, v);
        } else {
#pragma unroll
          for (int q = 0; q < V; ++q) v[q] = 0.0f;
        }
      }
      if (c < W) keep_total(c, v);
      const Chunk<T, V> w = c < W ? Chunk<T, V>::load(weight + c, W - c) : Chunk<T, V>::zero();
      if constexpr (MODE == kPlain) {
        if (c < W) {
          Chunk<T, V> a;
#pragma unroll
          for (int q = 0; q < V; ++q) a.v[q] = T(v[q] * rho * float(w.v[q]));
          a.store(y + row * W + c, W - c);
        }
      } else {
        // The 128 columns of a scale are 128 / V neighbouring lanes of a step.  rho
        // cancels in y / scale = 448 h w / max|h w|, which is formed in fp64 (h w is
        // exact there) and rounded to fp32 and then to 8 bits: a code differs from the exact
        // one only where h's own rounding or that one crosses the border of two codes.
        double out[V], top = 0.0;
#pragma unroll
        for (int q = 0; q < V; ++q) {
          out[q] = double(v[q]) * double(float(w.v[q]));
          top = fmax(top, fabs(out[q]));
        }
#pragma unroll
        for (int m = 1; m < kScaleGroup / V; m *= 2) top = fmax(top, __shfl_xor(top, m));
        if (c < W) {
          const float scale = float(top * double(rho)) / kLargest8;
          if (c % kScaleGroup == 0) scales[row * groups + c / kScaleGroup] = scale;
          // columns of zeros have scale 0 and codes 0; what is not a number stays so
          const double per = scale > 0.0f ? double(kLargest8) / top : double(scale);
          uint32_t packed[V / 4];
#pragma unroll
          for (int q = 0; q < V / 4; ++q) {
            int word = 0;
            word = __builtin_amdgcn_cvt_pk_fp8_f32(float(out[4 * q] * per), float(out[4 * q + 1] * per), word, false);
            word = __builtin_amdgcn_cvt_pk_fp8_f32(float(out[4 * q + 2] * per), float(out[4 * q + 3] * per), word, true);
            packed[q] = uint32_t(word);
          }
          Chunk<uint8_t, V> a;
#pragma unroll
          for (int q = 0; q < V; ++q) a.v[q] = uint8_t(packed[q / 4] >> (8 * (q % 4)));
          a.store(codes + row * W + c, W - c);
        }
      }
    }
  }
}

// The gradient: a workgroup walks over rows and keeps its sums of the weight's
// gradient, a lane those of its own columns; they are added over the
// workgroup's groups and written as one of `gridDim.x` partial rows, which
// rms_norm_weight_kernel adds in order.  The next row is read while the present
// one is summed: a row is one round trip to memory and two sums over lanes, and by
// itself that is all a wave does.  800 000 x 161 fp32: 750 -> 480 us for 2.06 GB.
// K = 0: the row is read twice and the sums stand in the workgroup's own partial
// row in memory, where each column belongs to one lane.
template <typename T, int L, int K>
__global__ __launch_bounds__(kThreads) void rms_norm_adjoint_kernel(const T* __restrict__ adjoint,
                                                                    const T* __restrict__ total_adjoint,
                                                                    const T* __restrict__ total,
                                                                    const T* __restrict__ weight, int64_t rows, int W,
                                                                    float epsilon, T* __restrict__ dx,
                                                                    float* __restrict__ partial) {
  constexpr int V = kChunk<T>;
  constexpr int H = K > 0 ? K : 1;
  constexpr int per = kThreads / L;
  typedef Chunk<T, V> C;
  __shared__ float part[2 * kThreads / 64];
  __shared__ float shared_dw[K > 0 && per > 1 ? L * K * V : 1];
  const int lane = int(threadIdx.x) % L;
  const int group = int(threadIdx.x) / L;
  float* mine = partial + int64_t(blockIdx.x) * W;
  const int64_t step = int64_t(gridDim.x) * per;
  int64_t row = int64_t(blockIdx.x) * per + group;
  if constexpr (K > 0) {
    struct RowOf {
      C h[H], g[H], t[H];
    };
    C w[H];
    float dw[H][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * L + lane) * V;
      w[k] = c < W ? C::load(weight + c, W - c) : C::zero();
#pragma unroll
      for (int q = 0; q < V; ++q) dw[k][q] = 0.0f;
    }
    auto read = [&](int64_t r) {
      RowOf x;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * L + lane) * V;
        x.h[k] = c < W ? C::load(total + r * W + c, W - c) : C::zero();
        x.g[k] = c < W ? C::load(adjoint + r * W + c, W - c) : C::zero();
        x.t[k] = c < W && total_adjoint ? C::load(total_adjoint + r * W + c, W - c) : C::zero();
      }
      return x;
    };
    RowOf next;
    if (row < rows) next = read(row);
    for (; row < rows; row += step) {
      const RowOf x = next;
      if (row + step < rows) next = read(row + step);
      float square = 0.0f, along = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float h = float(x.h[k].v[q]);
          square += h * h;
          along += h * (float(x.g[k].v[q]) * float(w[k].v[q]));
        }
      row_sums<L>(square, along, part);
      const float rho = 1.0f / sqrtf(square / float(W) + epsilon);
      const float pull = along / float(W) * rho * rho;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * L + lane) * V;
        C a;
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float h = float(x.h[k].v[q]), g = float(x.g[k].v[q]);
          a.v[q] = T(rho * (g * float(w[k].v[q]) - h * pull) + float(x.t[k].v[q]));
          dw[k][q] += g * h * rho;
        }
        if (c < W) a.store(dx + row * W + c, W - c);
      }
    }
    // groups in turn, so that the order of the sums is fixed
    for (int turn = 0; turn < per; ++turn) {
      if (group == turn) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (k * L + lane) * V;
#pragma unroll
          for (int q = 0; q < V; ++q) {
            if (per > 1) {
              float& s = shared_dw[c + q];
              s = turn == 0 ? dw[k][q] : s + dw[k][q];
              if (turn == per - 1 && c + q < W) mine[c + q] = s;
            } else if (c + q < W) {
              mine[c + q] = dw[k][q];
            }
          }
        }
      }
      if (per > 1) __syncthreads();
    }
  } else {
    for (int c = threadIdx.x; c < W; c += kThreads) mine[c] = 0.0f;
    __syncthreads();
    for (; row < rows; row += step) {
      float square = 0.0f, along = 0.0f;
      for (int c = lane * V; c < W; c += L * V) {
        const C h = C::load(total + row * W + c, W - c), g = C::load(adjoint + row * W + c, W - c),
                w = C::load(weight + c, W - c);
#pragma unroll
        for (int q = 0; q < V; ++q) {
          square += float(h.v[q]) * float(h.v[q]);
          along += float(h.v[q]) * (float(g.v[q]) * float(w.v[q]));
        }
      }
      row_sums<L>(square, along, part);
      const float rho = 1.0f / sqrtf(square / float(W) + epsilon);
      const float pull = along / float(W) * rho * rho;
      for (int c = lane * V; c < W; c += L * V) {
        const C hc = C::load(total + row * W + c, W - c), gc = C::load(adjoint + row * W + c, W - c),
                w = C::load(weight + c, W - c);
        const C t = total_adjoint ? C::load(total_adjoint + row * W + c, W - c) : C::zero();
        C a;
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float h = float(hc.v[q]), g = float(gc.v[q]);
          a.v[q] = T(rho * (g * float(w.v[q]) - h * pull) + float(t.v[q]));
          if (c + q < W) mine[c + q] += g * h * rho;
        }
        a.store(dx + row * W + c, W - c);
      }
    }
  }
}

// dw[c] = sum of the partial rows' column c: a lane a column, sixteen waves
// over the rows, their sums added in order.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_weight_kernel(const float* __restrict__ partial, int count, int W,
                                                               T* __restrict__ dw) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = int(blockIdx.x) * 64 + lane;
  float s = 0.0f;
  if (c < W) {
    for (int p0 = wave; p0 < count; p0 += 16 * 8) {  // eight loads in flight
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = p0 + 16 * k < count ? partial[int64_t(p0 + 16 * k) * W + c] : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < W) {
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += sums[w][lane];
    dw[c] = T(t);
  }
}

// Workgroups that fill the card: eight of four waves in a compute unit.
inline int resident_groups(int64_t wanted) { return int(wanted < 2048 ? (wanted < 1 ? 1 : wanted) : 2048); }

// Partial rows of the weight's gradient, a workgroup each: eight workgroups a
// compute unit, four for wide rows, whose partial rows would be a larger part of the traffic and
// whose lanes have more in flight.
inline int partial_rows(int64_t rows, int per, int64_t width) {
  const int64_t n = (rows + per - 1) / per, most = width <= 512 ? 2048 : 1024;
  return int(n < most ? (n < 1 ? 1 : n) : most);
}

struct Shape {
  int L, K;
};

// The group and the chunks of a row of `width` values: the smallest group that
// holds it in at most eight chunks of 16 bytes a lane (four for the gradient,
// which keeps three values for each); 0 chunks where 256 lanes do not.  Rows too few
// for a wave on every SIMD are latency, and take four waves if one would hold more than a
// chunk a lane: 37 rows of 4 096 in bf16, 8 bits, 11.6 us by one wave, 5.1 by four.
constexpr int64_t kFewRows = 1024;

inline Shape shape_of(int64_t rows, int width, int V, int most, int least) {
  const int lanes[4] = {4, 16, 64, 256};
  for (int i = 0; i < 4; ++i) {
    if (lanes[i] < least) continue;
    const int limit = lanes[i] < 64 ? 2 : lanes[i] == 64 && rows <= kFewRows ? 1 : most;
    const int k = (width + lanes[i] * V - 1) / (lanes[i] * V);
    if (k <= limit) return {lanes[i], k <= 1 ? 1 : k <= 2 ? 2 : k <= 4 ? 4 : 8};
  }
  return {256, 0};
}

template <typename T, int L, int K, int MODE>
int forward_as(const void* x, const void* r, const void* w, int64_t rows, int W, float eps, void* total, void* y,
               void* codes, void* scales, hipStream_t s) {
  constexpr int per = kThreads / L;
  const dim3 grid(resident_groups((rows + per - 1) / per));
  hipLaunchKernelGGL((rms_norm_kernel<T, L, K, MODE>), grid, dim3(kThreads), 0, s, static_cast<const T*>(x),
                     static_cast<const T*>(r), static_cast<const T*>(w), rows, W, eps, static_cast<T*>(total),
                     static_cast<T*>(y), static_cast<uint8_t*>(codes), static_cast<float*>(scales));
  return check_launch("rms_norm_kernel");
}

template <typename T, int MODE, typename... A>
int forward_shaped(Shape sh, A... a) {
  if constexpr (MODE == kPlain) {
    if (sh.L == 4) return sh.K == 1 ? forward_as<T, 4, 1, MODE>(a...) : forward_as<T, 4, 2, MODE>(a...);
    if (sh.L == 16) return sh.K == 1 ? forward_as<T, 16, 1, MODE>(a...) : forward_as<T, 16, 2, MODE>(a...);
  }
  if (sh.L == 64) {
    if (sh.K == 1) return forward_as<T, 64, 1, MODE>(a...);
    if (sh.K == 2) return forward_as<T, 64, 2, MODE>(a...);
    if (sh.K == 4) return forward_as<T, 64, 4, MODE>(a...);
    return forward_as<T, 64, 8, MODE>(a...);
  }
  if (sh.K == 1) return forward_as<T, 256, 1, MODE>(a...);
  if (sh.K == 2) return forward_as<T, 256, 2, MODE>(a...);
  if (sh.K == 4) return forward_as<T, 256, 4, MODE>(a...);
  if (sh.K == 8) return forward_as<T, 256, 8, MODE>(a...);
  return forward_as<T, 256, 0, MODE>(a...);
}

template <typename T, int L, int K>
int adjoint_as(const void* g, const void* tg, const void* h, const void* w, int64_t rows, int W, float eps, void* dx,
               void* dw, void* workspace, hipStream_t s) {
  const int count = partial_rows(rows, kThreads / L, W);
  float* partial = static_cast<float*>(workspace);
  hipLaunchKernelGGL((rms_norm_adjoint_kernel<T, L, K>), dim3(count), dim3(kThreads), 0, s, static_cast<const T*>(g),
                     static_cast<const T*>(tg), static_cast<const T*>(h), static_cast<const T*>(w), rows, W, eps,
                     static_cast<T*>(dx), partial);
  if (int rc = check_launch("rms_norm_adjoint_kernel")) return rc;
  hipLaunchKernelGGL((rms_norm_weight_kernel<T>), dim3((W + 63) / 64), dim3(1024), 0, s, partial, count, W,
                     static_cast<T*>(dw));
  return check_launch("rms_norm_weight_kernel");
}

template <typename T, typename... A>
int adjoint_shaped(Shape sh, A... a) {
  if (sh.L == 4) return sh.K == 1 ? adjoint_as<T, 4, 1>(a...) : adjoint_as<T, 4, 2>(a...);
  if (sh.L == 16) return sh.K == 1 ? adjoint_as<T, 16, 1>(a...) : adjoint_as<T, 16, 2>(a...);
  if (sh.L == 64) {
    if (sh.K == 1) return adjoint_as<T, 64, 1>(a...);
    if (sh.K == 2) return adjoint_as<T, 64, 2>(a...);
    return adjoint_as<T, 64, 4>(a...);
  }
  if (sh.K == 1) return adjoint_as<T, 256, 1>(a...);
  if (sh.K == 2) return adjoint_as<T, 256, 2>(a...);
  if (sh.K == 4) return adjoint_as<T, 256, 4>(a...);
  return adjoint_as<T, 256, 0>(a...);
}

int check_norm(int dtype, int64_t rows, int64_t width, double epsilon) {
  YE3T_REQUIRE(rows >= 0 && width >= 1, "rows and width must be positive");
  YE3T_REQUIRE(width <= (1 << 24), "rows of more than 2^24 values are not supported");
  YE3T_REQUIRE(epsilon > 0.0, "epsilon must be positive");
  if (dtype != YE3T_F32 && dtype != YE3T_BF16)
    return set_error(YE3T_EDTYPE, "unsupported dtype %d; expected float32 or bfloat16", dtype);
  return YE3T_OK;
}

// fp32's smallest normal value at least: rows of zeros divide by its root.
inline float held_epsilon(double epsilon) { return epsilon < 1.17549435e-38 ? 1.17549435e-38f : float(epsilon); }

inline Shape adjoint_shape(int dtype, int64_t rows, int64_t width) {
  return shape_of(rows, int(width), dtype == YE3T_F32 ? kChunk<float> : kChunk<__bf16>, 4, 1);
}

}  // namespace
}  // namespace ye3t

using namespace ye3t;

extern "C" {

int ye3t_hip_rms_norm(int dtype, const void* x, const void* residual, const void* weight, int64_t rows, int64_t width,
                      double epsilon, void* total, void* y, ye3t_stream_t stream) {
  clear_error();
  if (int rc = check_norm(dtype, rows, width, epsilon)) return rc;
  if (rows == 0) return YE3T_OK;
  YE3T_REQUIRE(x && weight && y, "the norm needs rows, a weight and an output");
  YE3T_REQUIRE(!residual || total, "a residual needs an output for the sum");
  const int W = int(width);
  const float eps = held_epsilon(epsilon);
  void* none = nullptr;
  if (dtype == YE3T_F32)
    return forward_shaped<float, kPlain>(shape_of(rows, W, kChunk<float>, 8, 1), x, residual, weight, rows, W, eps, total, y,
                                         none, none, as_stream(stream));
  return forward_shaped<__bf16, kPlain>(shape_of(rows, W, kChunk<__bf16>, 8, 1), x, residual, weight, rows, W, eps, total, y,
                                        none, none, as_stream(stream));
}

int ye3t_hip_rms_norm_8bit(int dtype, const void* x, const void* residual, const void* weight, int64_t rows,
                           int64_t width, double epsilon, void* total, void* codes, void* scales,
                           ye3t_stream_t stream) {
  clear_error();
  if (int rc = check_norm(dtype, rows, width, epsilon)) return rc;
  if (rows == 0) return YE3T_OK;
  YE3T_REQUIRE(x && weight && codes && scales, "the norm needs rows, a weight, codes and scales");
  YE3T_REQUIRE(!residual || total, "a residual needs an output for the sum");
  const int W = int(width);
  const float eps = held_epsilon(epsilon);
  void* none = nullptr;
  // a scale's 128 columns lie in one wave: 32 lanes in fp32
  if (dtype == YE3T_F32)
    return forward_shaped<float, kEightBit>(shape_of(rows, W, kChunk<float>, 8, 64), x, residual, weight, rows, W, eps, total,
                                            none, codes, scales, as_stream(stream));
  return forward_shaped<__bf16, kEightBit>(shape_of(rows, W, kChunk<__bf16>, 8, 64), x, residual, weight, rows, W, eps, total,
                                           none, codes, scales, as_stream(stream));
}

int64_t ye3t_hip_rms_norm_adjoint_workspace_bytes(int dtype, int64_t rows, int64_t width) {
  clear_error();
  if (check_norm(dtype, rows, width, 1.0)) return -1;
  return int64_t(partial_rows(rows, kThreads / adjoint_shape(dtype, rows, width).L, width)) * width * int64_t(sizeof(float));
}

int ye3t_hip_rms_norm_adjoint(int dtype, const void* adjoint, const void* total_adjoint, const void* total,
                              const void* weight, int64_t rows, int64_t width, double epsilon, void* x_adjoint,
                              void* weight_adjoint, void* workspace, int64_t workspace_bytes, ye3t_stream_t stream) {
  clear_error();
  if (int rc = check_norm(dtype, rows, width, epsilon)) return rc;
  YE3T_REQUIRE(weight && weight_adjoint, "the gradient needs the weight and an output for its gradient");
  YE3T_REQUIRE(rows == 0 || (adjoint && total && x_adjoint), "the gradient needs the adjoint, the sum and an output");
  YE3T_REQUIRE(workspace && workspace_bytes >= ye3t_hip_rms_norm_adjoint_workspace_bytes(dtype, rows, width),
               "the workspace is smaller than ye3t_hip_rms_norm_adjoint_workspace_bytes");
  const Shape sh = adjoint_shape(dtype, rows, width);
  const int W = int(width);
  const float eps = held_epsilon(epsilon);
  if (dtype == YE3T_F32)
    return adjoint_shaped<float>(sh, adjoint, total_adjoint, total, weight, rows, W, eps, x_adjoint, weight_adjoint,
                                 workspace, as_stream(stream));
  return adjoint_shaped<__bf16>(sh, adjoint, total_adjoint, total, weight, rows, W, eps, x_adjoint, weight_adjoint,
                                workspace, as_stream(stream));
}

}  // extern "C"
