// y = residual + dropout(x), and its gradient, which is the same without a residual.
//
// A lane takes eight columns of a row, one call of the generator, and two such chunks at a time.  Bound by
// memory: 200 000 x 513 in bf16, rows that start at any multiple of two bytes, 138 us with a residual (4.5 TB/s) and 91
// without; the generator's twenty products a call take about a third of that.
#include "random.h"
#include "rows.h"

namespace ye3t {
namespace {

constexpr int kThreads = 256;

template <typename T, bool ADD>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                           int64_t rows, int W, int chunks, Dropout d,
                                                           T* __restrict__ y) {
  constexpr int STEPS = 2;
  const int64_t all = rows * chunks;
  const uint64_t seed = seed_of(d);
  for (int64_t i0 = int64_t(blockIdx.x) * (kThreads * STEPS); i0 < all; i0 += int64_t(gridDim.x) * (kThreads * STEPS)) {
    Chunk<T, 8> a[STEPS], r[STEPS];
    int64_t row[STEPS];
    int c[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int64_t i = i0 + k * kThreads + threadIdx.x;
      row[k] = all <= INT32_MAX ? int64_t(uint32_t(i) / uint32_t(chunks)) : i / chunks;
      c[k] = int(i - row[k] * chunks) * 8;
      if (i < all) {
        a[k] = Chunk<T, 8>::load(x + row[k] * W + c[k], W - c[k]);
        if (ADD) r[k] = Chunk<T, 8>::load(residual + row[k] * W + c[k], W - c[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (i0 + k * kThreads + threadIdx.x >= all) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = float(a[k].v[q]);
      drop(d, seed, row[k], uint32_t(c[k]) / 8, v);
      Chunk<T, 8> out;
#pragma unroll
      for (int q = 0; q < 8; ++q) out.v[q] = T(ADD ? v[q] + float(r[k].v[q]) : v[q]);
      out.store(y + row[k] * W + c[k], W - c[k]);
    }
  }
}

template <typename T>
int launch(const void* x, const void* residual, int64_t rows, int64_t width, const Dropout& d, void* y, hipStream_t s) {
  const int64_t chunks = (width + 7) / 8;
  int64_t groups = (rows * chunks + 2 * kThreads - 1) / (2 * kThreads);
  if (groups > (1 << 20)) groups = 1 << 20;
  hipLaunchKernelGGL((residual ? dropout_kernel<T, true> : dropout_kernel<T, false>), dim3(unsigned(groups)),
                     dim3(kThreads), 0, s, static_cast<const T*>(x), static_cast<const T*>(residual), rows, int(width),
                     int(chunks), d, static_cast<T*>(y));
  return check_launch("dropout_kernel");
}

}  // namespace
}  // namespace ye3t

using namespace ye3t;

extern "C" int ye3t_hip_dropout(int dtype, const void* x, const void* residual, int64_t rows, int64_t width,
                                int64_t below, uint32_t layer, uint64_t seed, const int64_t* device_seed, void* y,
                                ye3t_stream_t stream) {
  clear_error();
  YE3T_REQUIRE(rows >= 0 && rows <= INT64_MAX / 4 / (width > 0 ? width : 1) && width >= 0 && width <= (1 << 24),
               "dropout takes rows of up to 2^24 values");
  YE3T_REQUIRE(below >= 0 && below <= 65536, "the dropped share must be 0 .. 65536");
  if (dtype != YE3T_F32 && dtype != YE3T_BF16)
    return set_error(YE3T_EDTYPE, "unsupported dtype %d; expected float32 or bfloat16", dtype);
  if (rows == 0 || width == 0) return YE3T_OK;
  YE3T_REQUIRE(x && y, "dropout needs rows and an output");
  const Dropout d = dropout_of(below, layer, seed, device_seed);
  return dtype == YE3T_F32 ? launch<float>(x, residual, rows, width, d, y, as_stream(stream))
                           : launch<__bf16>(x, residual, rows, width, d, y, as_stream(stream));
}
