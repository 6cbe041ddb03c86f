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

// dz in the workspace and the sums of the shares behind it; the same whatever the adjoint's address is.
int64_t dz_bytes(const ye3t_linear_args& a) {
  return shaped(a) ? up(a.rows * a.outputs * (a.dtype == YE3T_F32 ? 4 : 2)) : 0;
}
// dx and dW are made one after the other: what one takes for its parts the other takes after it.
int64_t adjoint_bytes(const ye3t_linear_args& a) {
  const int64_t parts = a.dtype == YE3T_F32 ? row_bytes(backward_of<float>(a, nullptr))
                                            : row_bytes(backward_of<__bf16>(a, nullptr));
  const int64_t shares = a.dtype == YE3T_F32 ? weight_bytes(weights_of<float>(a, nullptr))
                                             : weight_bytes(weights_of<__bf16>(a, nullptr));
  return dz_bytes(a) + (shares > parts ? shares : parts) + 256;
}

template <typename T>
int adjoint_as(const ye3t_linear_args& a, const void* adjoint, const void* kept, void* input_adjoint,
               void* weight_adjoint, void* bias_adjoint, char* work, hipStream_t s) {
  const T* dz = static_cast<const T*>(adjoint);
  if (shaped(a) && a.rows > 0 && a.outputs > 0) {
    T* to = reinterpret_cast<T*>(work);
    const int64_t chunks = (a.outputs + 7) / 8;
    int64_t groups = (a.rows * chunks + kThreads - 1) / kThreads;
    if (groups > (1 << 20)) groups = 1 << 20;
    hipLaunchKernelGGL((epilogue_adjoint_kernel<T>), dim3(unsigned(groups)), dim3(kThreads), 0, s, dz,
                       static_cast<const T*>(kept), a.rows, int(a.outputs), int(chunks), a.activation,
                       dropout_of(a.drop_below, a.layer, a.seed, a.device_seed), to);
    if (int rc = check_launch("epilogue_adjoint_kernel")) return rc;
    dz = to;
  }
  if (input_adjoint) {
    RowProduct<T> p = backward_of(a, dz);
    p.out = static_cast<T*>(input_adjoint);
    if (int rc = launch_rows(p, work + dz_bytes(a), s)) return rc;
  }
  if (weight_adjoint || bias_adjoint) {
    WeightProduct<T> p = weights_of<T>(a, dz);
    p.out = static_cast<T*>(weight_adjoint);
    p.sums = static_cast<T*>(bias_adjoint);
    if (int rc = launch_weights(p, work + dz_bytes(a), s)) return rc;
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

int64_t ye3t_hip_linear_adjoint_workspace_bytes(const ye3t_linear_args* args) {
  clear_error();
  if (!args) return set_error(YE3T_EINVAL, "the product needs its arguments");
  if (linear::check_linear(*args)) return -1;
  return linear::adjoint_bytes(*args);
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
  YE3T_REQUIRE(workspace && workspace_bytes >= linear::adjoint_bytes(*args),
               "the workspace is smaller than ye3t_hip_linear_adjoint_workspace_bytes");
  char* work = static_cast<char*>(workspace);
  return args->dtype == YE3T_F32
             ? linear::adjoint_as<float>(*args, adjoint, preactivation, input_adjoint, weight_adjoint, bias_adjoint, work,
                                         as_stream(stream))
             : linear::adjoint_as<__bf16>(*args, adjoint, preactivation, input_adjoint, weight_adjoint, bias_adjoint, work,
                                          as_stream(stream));
}

}  // extern "C"
