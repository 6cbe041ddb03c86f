// Entry points of the products with learned weights, and the epilogue's gradient.
#include "linear.h"

namespace ye3t {
namespace linear {
namespace {

constexpr int kThreads = 256;

// dz = D(g act'(z)), rounded to the storage type for the matrix instructions of both products that read it.  Dropped last:
// a dropped value is zero whatever its slope is, which is no number where its preactivation is none or infinite.  A
// kernel of its own, as both take dz straight to LDS.  A lane takes eight columns of a row.  Bound by memory: 16 384 x
// 4 096 in bf16 with gelu 82 us, 4.9 TB/s.
template <typename T>
__global__ __launch_bounds__(kThreads) void epilogue_adjoint_kernel(const T* __restrict__ adjoint,
                                                                    const T* __restrict__ kept, int64_t rows, int N,
                                                                    int chunks, int activation, Dropout d,
                                                                    T* __restrict__ dz) {
  const int64_t all = rows * chunks;
  const uint64_t seed = d.below ? seed_of(d) : 0;
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < all; i += int64_t(gridDim.x) * kThreads) {
    const int64_t row = all <= INT32_MAX ? int64_t(uint32_t(i) / uint32_t(chunks)) : i / chunks;
    const int n = int(i - row * chunks) * 8, left = N - n;
    const Chunk<T, 8> g = Chunk<T, 8>::load(adjoint + row * N + n, left);
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = float(g.v[q]);
    if (activation != kNone) {
      const Chunk<T, 8> z = Chunk<T, 8>::load(kept + row * N + n, left);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = through(activation, v[q], float(z.v[q]));
    }
    if (d.below) drop(d, seed, row, uint32_t(n) / 8, v);
    Chunk<T, 8> out;
#pragma unroll
    for (int q = 0; q < 8; ++q) out.v[q] = T(v[q]);
    out.store(dz + row * N + n, left);
  }
}

// The same in bf16 with the bias's gradient, summed of dz before it is rounded: it is a sum and takes no matrix instruction
// (16 384 x 4 096, gelu: 1.7e-3 from 64 bits, the last rounding; of the rounded dz 2.4e-3).  A workgroup goes through a share of
// one group's rows, `across` lanes of eight columns and the others down the rows, two rows of a lane in flight; shares of a group
// that has several leave their sums in fp32, and a second kernel adds them in order.  78 us at that size, and 4 for the join.
struct BiasSums {
  int64_t groups;
  bool grouped;
  const int32_t* order;
  const int64_t* offsets;
  int across;           // a power of two
  unsigned columns;     // workgroups along the columns
  int64_t share;
  __bf16* sums;         // [groups][N]
  float* part;          // [part_count(rows, share)][N]
};

__global__ __launch_bounds__(kThreads) void epilogue_adjoint_sums_kernel(const __bf16* __restrict__ adjoint,
                                                                         const __bf16* __restrict__ kept, int64_t rows,
                                                                         int N, int activation, Dropout d, BiasSums b,
                                                                         __bf16* __restrict__ dz) {
  constexpr int STEPS = 2;
  __shared__ float held[kThreads * 8];
  const int64_t slot = blockIdx.x / b.columns;
  const int column = int(threadIdx.x) & (b.across - 1), line = int(threadIdx.x) / b.across, down = kThreads / b.across;
  const int n0 = int(blockIdx.x % b.columns) * b.across * 8, n = n0 + column * 8, left = N - n;
  int64_t group = 0, begin = 0, first = slot * b.share, length = rows;
  if (b.grouped) {
    auto bound = [&](int64_t g) { return clamped(b.offsets[g], rows) / b.share + g; };
    group = find_owner(b.groups, slot, bound);
    first = (slot - bound(group)) * b.share;
    begin = clamped(b.offsets[group], rows);
    length = clamped(b.offsets[group + 1], rows) - begin;
  }
  if (first && first >= length) return;  // the first share of a group without rows writes its zeros
  const int64_t row0 = begin + first, rest = length - first;
  const int live = int(rest < 0 ? 0 : rest < b.share ? rest : b.share);
  const uint64_t seed = d.below ? seed_of(d) : 0;
  float sum[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) sum[q] = 0.0f;
  for (int k0 = line; left > 0 && k0 < live; k0 += STEPS * down) {
    Chunk<__bf16, 8> g[STEPS], z[STEPS];
    int64_t row[STEPS];
#pragma unroll
    for (int e = 0; e < STEPS; ++e) {
      const int k = k0 + e * down;
      row[e] = k < live ? row_at(b.order, row0 + k, rows) : -1;
      if (row[e] < 0) continue;
      g[e] = Chunk<__bf16, 8>::load(adjoint + row[e] * N + n, left);
      if (activation != kNone) z[e] = Chunk<__bf16, 8>::load(kept + row[e] * N + n, left);
    }
#pragma unroll
    for (int e = 0; e < STEPS; ++e) {
      if (row[e] < 0) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = float(g[e].v[q]);
      if (activation != kNone) {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = through(activation, v[q], float(z[e].v[q]));
      }
      if (d.below) drop(d, seed, row[e], uint32_t(n) / 8, v);
      Chunk<__bf16, 8> out;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        sum[q] += v[q];
        out.v[q] = __bf16(v[q]);
      }
      out.store(dz + row[e] * N + n, left);
    }
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) held[int(threadIdx.x) * 8 + q] = sum[q];
  __syncthreads();
  const int c = int(threadIdx.x);
  if (c >= b.across * 8 || n0 + c >= N) return;
  float s = 0.0f;
#pragma unroll 16
  for (int k = 0; k < down; ++k) s += held[k * b.across * 8 + c];
  if (length <= b.share) b.sums[group * N + n0 + c] = __bf16(s);
  else b.part[(part_of(begin, b.share) + first / b.share) * N + n0 + c] = s;
}

// A lane a column of a group that has several shares, sixteen lanes its shares
__global__ __launch_bounds__(kThreads) void bias_join_kernel(BiasSums b, int64_t rows, int N) {
  constexpr int COLUMNS = 16, DOWN = kThreads / COLUMNS;
  __shared__ float held[DOWN][COLUMNS];
  const int column = int(threadIdx.x) % COLUMNS, line = int(threadIdx.x) / COLUMNS, n = int(blockIdx.x) * COLUMNS + column;
  for (int64_t g = blockIdx.y; g < (b.grouped ? b.groups : 1); g += gridDim.y) {
    const int64_t begin = b.grouped ? clamped(b.offsets[g], rows) : 0;
    const int64_t length = (b.grouped ? clamped(b.offsets[g + 1], rows) : rows) - begin;
    if (length <= b.share) continue;  // the same for all lanes
    const float* from = b.part + part_of(begin, b.share) * N + n;
    const int shares = int((length + b.share - 1) / b.share);
    float s = 0.0f;
    if (n < N) {
#pragma unroll 8
      for (int k = line; k < shares; k += DOWN) s += from[int64_t(k) * N];
    }
    held[line][column] = s;
    __syncthreads();
    if (line == 0 && n < N) {
#pragma unroll
      for (int k = 1; k < DOWN; ++k) s += held[k][column];
      b.sums[g * N + n] = __bf16(s);
    }
    __syncthreads();
  }
}

// Shares that make about 4 096 workgroups, 512 at most of one group for the join, of a lane's two rows at least.  Sixteen
// lanes across and these shares: 16 384 x 4 096 78 us, by eight and half as many workgroups 94; 2 000 x 512 7 and 14.
BiasSums bias_sums(const ye3t_linear_args& a) {
  BiasSums b{};
  b.grouped = a.groups_given != 0;
  b.groups = a.groups;
  b.order = b.grouped ? a.order : nullptr;
  b.offsets = b.grouped ? a.offsets : nullptr;
  for (b.across = 1; b.across < 16 && b.across * 8 < a.outputs; b.across *= 2) {}
  b.columns = unsigned((a.outputs + b.across * 8 - 1) / (b.across * 8));
  const int64_t all = (a.rows * b.columns + 4095) / 4096, most = (a.rows + 511) / 512, least = 2 * kThreads / b.across;
  b.share = all > most ? all : most;
  if (b.share < least) b.share = least;
  if (b.share > (1 << 30)) b.share = 1 << 30;
  return b;
}

int check_linear(const ye3t_linear_args& a) {
  constexpr int64_t most = (int64_t(1) << 31) - 256;
  YE3T_REQUIRE(a.rows >= 0 && a.inputs >= 0 && a.outputs >= 0 && a.groups >= 0, "sizes must not be negative");
  if (a.dtype != YE3T_F32 && a.dtype != YE3T_BF16)
    return set_error(YE3T_EDTYPE, "unsupported dtype %d; expected float32 or bfloat16", a.dtype);
  YE3T_REQUIRE(a.rows < most && a.inputs <= (1 << 24) && a.outputs <= (1 << 24) && a.groups < (1 << 24),
               "at most 2^31 - 257 rows, 2^24 columns and 2^24 - 1 species");
  YE3T_REQUIRE(a.activation >= kNone && a.activation <= kGelu, "unknown activation %d", a.activation);
  YE3T_REQUIRE(a.drop_below >= 0 && a.drop_below <= 65536, "the dropped share must be 0 .. 65536");
  return YE3T_OK;
}

int check_pointers(const ye3t_linear_args& a) {
  const bool rows = a.rows > 0 && a.inputs > 0;
  YE3T_REQUIRE(!rows || a.input, "the product needs its input");
  YE3T_REQUIRE(a.inputs == 0 || a.outputs == 0 || a.weight || (a.groups_given && a.groups == 0),
               "the product needs its weight");
  YE3T_REQUIRE(!a.groups_given || (a.offsets && (a.rows == 0 || a.order)), "grouped rows need their order and offsets");
  YE3T_REQUIRE(a.input_row_stride >= 0 && a.weight_group_stride >= 0 && a.weight_row_stride >= 0,
               "strides must not be negative");
  return YE3T_OK;
}

template <typename T>
RowProduct<T> rows_of(const ye3t_linear_args& a) {
  RowProduct<T> p{};
  p.rows = a.rows;
  p.groups = a.groups;
  p.grouped = a.groups_given != 0;
  p.order = p.grouped ? a.order : nullptr;
  p.offsets = p.grouped ? a.offsets : nullptr;
  p.b = static_cast<const T*>(a.weight);
  p.b_group = a.weight_group_stride;
  p.b_row = a.weight_row_stride;
  return p;
}

template <typename T>
RowProduct<T> forward_of(const ye3t_linear_args& a) {
  RowProduct<T> p = rows_of<T>(a);
  p.a = static_cast<const T*>(a.input);
  p.a_row = a.input_row_stride;
  p.b_across = !a.turned;
  p.K = int(a.inputs);
  p.N = int(a.outputs);
  p.bias = static_cast<const T*>(a.bias);
  p.residual = static_cast<const T*>(a.residual);
  p.activation = a.activation;
  p.dropout = dropout_of(a.drop_below, a.layer, a.seed, a.device_seed);
  return p;
}

// dx = dz W^T
template <typename T>
RowProduct<T> backward_of(const ye3t_linear_args& a, const T* dz) {
  RowProduct<T> p = rows_of<T>(a);
  p.a = dz;
  p.a_row = a.outputs;
  p.b_across = a.turned != 0;
  p.K = int(a.outputs);
  p.N = int(a.inputs);
  return p;
}

template <typename T>
int forward_as(const ye3t_linear_args& a, void* kept, void* out, void* work, hipStream_t s) {
  RowProduct<T> p = forward_of<T>(a);
  p.kept = static_cast<T*>(kept);
  p.out = static_cast<T*>(out);
  return launch_rows(p, work, s);
}

int64_t forward_bytes(const ye3t_linear_args& a) {
  return a.dtype == YE3T_F32 ? row_bytes(forward_of<float>(a)) : row_bytes(forward_of<__bf16>(a));
}

inline bool shaped(const ye3t_linear_args& a) { return a.activation != kNone || a.drop_below > 0; }

// dW = x^T dz, or its transpose where the weight is kept turned
template <typename T>
WeightProduct<T> weights_of(const ye3t_linear_args& a, const T* dz) {
  WeightProduct<T> p{};
  const T* x = static_cast<const T*>(a.input);
  p.a = a.turned ? dz : x;
  p.b = a.turned ? x : dz;
  p.a_row = a.turned ? a.outputs : a.input_row_stride;
  p.b_row = a.turned ? a.input_row_stride : a.outputs;
  p.M = int(a.turned ? a.outputs : a.inputs);
  p.N = int(a.turned ? a.inputs : a.outputs);
  p.rows = a.rows;
  p.groups = a.groups;
  p.grouped = a.groups_given != 0;
  p.order = p.grouped ? a.order : nullptr;
  p.offsets = p.grouped ? a.offsets : nullptr;
  p.sums_of_a = a.turned != 0;
  return p;
}

// dz in the workspace, the bias's sums of its shares of rows behind it, and the sums of the products' shares behind those; the
// same whatever the adjoint's address is.
int64_t dz_bytes(const ye3t_linear_args& a) {
  return shaped(a) ? up(a.rows * a.outputs * (a.dtype == YE3T_F32 ? 4 : 2)) : 0;
}
int64_t bias_bytes(const ye3t_linear_args& a) {
  if (!shaped(a) || a.dtype == YE3T_F32 || a.rows == 0 || a.outputs == 0) return 0;
  return up(part_count(a.rows, bias_sums(a).share) * a.outputs * 4);
}
// dx and dW are made one after the other: what one takes for its parts the other takes after it.
int64_t adjoint_bytes(const ye3t_linear_args& a, bool input, bool weight, bool bias) {
  int64_t parts = 0, shares = 0;
  if (input)
    parts = a.dtype == YE3T_F32 ? row_bytes(backward_of<float>(a, nullptr)) : row_bytes(backward_of<__bf16>(a, nullptr));
  if (weight || bias)
    shares = a.dtype == YE3T_F32 ? weight_bytes(weights_of<float>(a, nullptr)) : weight_bytes(weights_of<__bf16>(a, nullptr));
  return dz_bytes(a) + (bias ? bias_bytes(a) : 0) + (shares > parts ? shares : parts) + 256;
}

template <typename T>
int launch_epilogue(const ye3t_linear_args& a, const T* adjoint, const T* kept, T* dz, hipStream_t s) {
  const int64_t chunks = (a.outputs + 7) / 8;
  int64_t groups = (a.rows * chunks + kThreads - 1) / kThreads;
  if (groups > (1 << 20)) groups = 1 << 20;
  hipLaunchKernelGGL((epilogue_adjoint_kernel<T>), dim3(unsigned(groups)), dim3(kThreads), 0, s, adjoint, kept, a.rows,
                     int(a.outputs), int(chunks), a.activation, dropout_of(a.drop_below, a.layer, a.seed, a.device_seed), dz);
  return check_launch("epilogue_adjoint_kernel");
}

int launch_epilogue_sums(const ye3t_linear_args& a, const __bf16* adjoint, const __bf16* kept, __bf16* dz, __bf16* sums,
                         void* part, hipStream_t s) {
  BiasSums b = bias_sums(a);
  b.sums = sums;
  b.part = static_cast<float*>(part);
  const int64_t slots = b.grouped ? a.rows / b.share + b.groups : (a.rows + b.share - 1) / b.share;
  if (!fits_grid(slots * b.columns, kThreads))
    return set_error(YE3T_EUNSUPPORTED, "biases of %lld for %lld species are too many for one launch", (long long)a.outputs,
                     (long long)a.groups);
  hipLaunchKernelGGL(epilogue_adjoint_sums_kernel, dim3(unsigned(slots * b.columns)), dim3(kThreads), 0, s, adjoint, kept,
                     a.rows, int(a.outputs), a.activation, dropout_of(a.drop_below, a.layer, a.seed, a.device_seed), b, dz);
  if (int rc = check_launch("epilogue_adjoint_sums_kernel")) return rc;
  if (a.rows <= b.share) return YE3T_OK;
  const int64_t groups = b.grouped ? b.groups : 1;
  hipLaunchKernelGGL(bias_join_kernel, dim3(unsigned((a.outputs + 15) / 16), unsigned(groups < 65535 ? groups : 65535)),
                     dim3(kThreads), 0, s, b, a.rows, int(a.outputs));
  return check_launch("bias_join_kernel");
}

template <typename T>
int adjoint_as(const ye3t_linear_args& a, const void* adjoint, const void* kept, void* input_adjoint,
               void* weight_adjoint, void* bias_adjoint, char* work, hipStream_t s) {
  const T* dz = static_cast<const T*>(adjoint);
  char* behind = work + dz_bytes(a) + (bias_adjoint ? bias_bytes(a) : 0);
  if (shaped(a) && a.rows > 0 && a.outputs > 0) {
    T* to = reinterpret_cast<T*>(work);
    bool summed = false;
    if constexpr (sizeof(T) == 2) {
      summed = bias_adjoint && (!a.groups_given || a.groups > 0);
      if (summed) {
        if (int rc = launch_epilogue_sums(a, dz, static_cast<const T*>(kept), to, static_cast<T*>(bias_adjoint),
                                          work + dz_bytes(a), s))
          return rc;
        bias_adjoint = nullptr;  // made
      }
    }
    if (!summed) {
      if (int rc = launch_epilogue(a, dz, static_cast<const T*>(kept), to, s)) return rc;
    }
    dz = to;
  }
  if (input_adjoint) {
    RowProduct<T> p = backward_of(a, dz);
    p.out = static_cast<T*>(input_adjoint);
    if (int rc = launch_rows(p, behind, s)) return rc;
  }
  if (weight_adjoint || bias_adjoint) {
    WeightProduct<T> p = weights_of<T>(a, dz);
    p.out = static_cast<T*>(weight_adjoint);
    p.sums = static_cast<T*>(bias_adjoint);
    if (int rc = launch_weights(p, behind, s)) return rc;
  }
  return YE3T_OK;
}

}  // namespace
}  // namespace linear
}  // namespace ye3t

using namespace ye3t;

extern "C" {

int64_t ye3t_hip_linear_workspace_bytes(const ye3t_linear_args* args) {
  clear_error();
  if (!args) return set_error(YE3T_EINVAL, "the product needs its arguments");
  if (linear::check_linear(*args)) return -1;
  return linear::forward_bytes(*args);
}

int ye3t_hip_linear(const ye3t_linear_args* args, void* preactivation, void* out, void* workspace,
                    int64_t workspace_bytes, ye3t_stream_t stream) {
  clear_error();
  YE3T_REQUIRE(args, "the product needs its arguments");
  if (int rc = linear::check_linear(*args)) return rc;
  if (args->rows == 0 || args->outputs == 0) return YE3T_OK;
  if (int rc = linear::check_pointers(*args)) return rc;
  YE3T_REQUIRE(out, "the product needs an output");
  const int64_t bytes = linear::forward_bytes(*args);
  YE3T_REQUIRE(bytes == 0 || (workspace && workspace_bytes >= bytes),
               "the workspace is smaller than ye3t_hip_linear_workspace_bytes");
  return args->dtype == YE3T_F32
             ? linear::forward_as<float>(*args, preactivation, out, workspace, as_stream(stream))
             : linear::forward_as<__bf16>(*args, preactivation, out, workspace, as_stream(stream));
}

int64_t ye3t_hip_linear_adjoint_workspace_bytes_of(const ye3t_linear_args* args, int input, int weight, int bias) {
  clear_error();
  if (!args) return set_error(YE3T_EINVAL, "the product needs its arguments");
  if (linear::check_linear(*args)) return -1;
  return linear::adjoint_bytes(*args, input, weight, bias);
}

int64_t ye3t_hip_linear_adjoint_workspace_bytes(const ye3t_linear_args* args) {
  return ye3t_hip_linear_adjoint_workspace_bytes_of(args, 1, 1, 1);
}

int ye3t_hip_linear_adjoint(const ye3t_linear_args* args, const void* adjoint, const void* preactivation,
                            void* input_adjoint, void* weight_adjoint, void* bias_adjoint, void* workspace,
                            int64_t workspace_bytes, ye3t_stream_t stream) {
  clear_error();
  YE3T_REQUIRE(args, "the product needs its arguments");
  if (int rc = linear::check_linear(*args)) return rc;
  if (int rc = linear::check_pointers(*args)) return rc;
  const bool any = args->rows > 0 && args->outputs > 0;
  YE3T_REQUIRE(!any || adjoint, "the gradient needs the output's adjoint");
  YE3T_REQUIRE(!any || args->activation == linear::kNone || preactivation,
               "the gradient of an activation needs the preactivation");
  YE3T_REQUIRE(!bias_adjoint || weight_adjoint || args->inputs == 0, "the bias's gradient comes with the weight's");
  YE3T_REQUIRE(workspace && workspace_bytes >= linear::adjoint_bytes(*args, input_adjoint, weight_adjoint, bias_adjoint),
               "the workspace is smaller than ye3t_hip_linear_adjoint_workspace_bytes");
  char* work = static_cast<char*>(workspace);
  return args->dtype == YE3T_F32
             ? linear::adjoint_as<float>(*args, adjoint, preactivation, input_adjoint, weight_adjoint, bias_adjoint, work,
                                         as_stream(stream))
             : linear::adjoint_as<__bf16>(*args, adjoint, preactivation, input_adjoint, weight_adjoint, bias_adjoint, work,
                                          as_stream(stream));
}

}  // extern "C"
