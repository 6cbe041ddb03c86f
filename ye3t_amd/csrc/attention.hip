// Atom attention: forward kernels, the sums of the gradients to slopes and
// positions, and the entry points.
#include "attention.h"

namespace ye3t {
namespace attention {
namespace {

// ---- forward -----------------------------------------------------------------
// One pass over the keys with the running maximum and sum of the softmax; the scores,
// their weights and the output rows stay in registers, so memory is read once for each 128 rows
// and written once.  NW waves of 32 rows, KT keys a tile.  SPLIT: grid axis z takes equal
// parts of each structure's key tiles and leaves its sums to attention_join_kernel.
//
// Bound by what a score costs beside the products: about 17 vector operations with
// distance and cap, four of them of quarter rate, 5 without.  8 192 atoms, 16
// heads of 128 over 4, bf16: 0.68 ms, 810 TFLOP/s (1 136 for a large product here), the
// matrix units busy for 34 % of the time and the vector units for 58 %; 96 structures of
// 480, 8 heads of 64, distances, cap and mask: 0.21 ms, 232 TFLOP/s.  fp32: 40 structures
// of 1 000, 8 heads of 64, distances: 0.98 ms, 87 of 152 TFLOP/s (matrix units 57 %, vector
// units 25 %).  One row against 9 000 atoms in 24 structures: 0.10 ms for 437 MB.
template <typename T, int DP, int NW, int KT, bool BIAS, Cap CAP, bool SPLIT>
__global__ __launch_bounds__(64 * NW, (kForwardWaves<T, DP, NW>)) void attention_kernel(Problem p, T* __restrict__ out, float* __restrict__ log_sums,
                                                            float* __restrict__ part, float* __restrict__ part_stats) {
  constexpr int TILE = 32 * NW, NU = DP / (2 * kChunk<T>), ND = DP / 32;
  constexpr int BUFFERS = NW == 1 ? 1 : 2;
  constexpr bool FRESH = NW == 1 && !SPLIT;
  __shared__ __align__(16) T ktiles[BUFFERS * KT * DP];
  __shared__ __align__(16) T vtiles[BUFFERS * KT * DP];
  __shared__ f32x4 places[BUFFERS * KT];
  const Item item = item_of(p.offsets, p.structures, p.queries, p.group, TILE, blockIdx.x);
  const Span own = span_of(p.offsets, item.structure, p.queries);
  const int64_t rows = int64_t(own.length) * p.group;
  if (item.first < 0 || item.first >= rows) return;
  const Span key = span_of(p.key_offsets, item.structure, p.keys);
  const int key_head = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const Row row = row_of(p, own.begin, item.first + 32 * wave + (lane & 31), rows, key_head);
  const bool busy = item.first + 32 * wave < rows;  // of the whole wave

  Op<T> q[NU];
  line_operand<T, DP>(row.exists ? static_cast<const T*>(p.q) + row.token * p.q_row + row.head * p.q_head : nullptr,
                      p.D, half, q);
  float x = 0.0f, y = 0.0f, z = 0.0f, slope = 0.0f;
  if (BIAS && row.exists) {
    x = p.positions[3 * row.token];
    y = p.positions[3 * row.token + 1];
    z = p.positions[3 * row.token + 2];
    slope = p.slopes[row.head] * kLog2e;
  }
  int tiles = (key.length + KT - 1) / KT, tile = 0;
  if (SPLIT) {
    const int each = (tiles + gridDim.z - 1) / gridDim.z;
    tile = int(blockIdx.z) * each;
    tiles = tile + each < tiles ? tile + each : tiles;
  }
  f32x16 acc[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) acc[t] = zeros();
  float top = -INFINITY, sum = 0.0f;
  KeyTiles<T, DP, KT, 64 * NW, BUFFERS, FRESH, BIAS> tiles_of{p,      key,    static_cast<const T*>(p.k) + key_head * p.k_head,
                                                       static_cast<const T*>(p.v) + key_head * p.v_head,
                                                       ktiles, vtiles, places};
  if (tile < tiles) tiles_of.start(tile);
  for (; tile < tiles; ++tile) {
    tiles_of.take(tile, tiles);
    const T *ktile = tiles_of.keys(tile), *vtile = tiles_of.values(tile);
    const f32x4* place = tiles_of.places_of(tile);
    if (!busy) continue;
    const unsigned now_lane = anew<FRESH>(lane) & 63;
    const bool masked = p.key_mask != nullptr || (tile + 1) * KT > key.length;
    f32x16 s[KT / 32];
    float high = -INFINITY;
#pragma unroll
    for (int n = 0; n < KT / 32; ++n) {
      s[n] = zeros();
      in_flight<NU>([&](int u) { return line_chunk<T, DP>(ktile, 32 * n + int(now_lane & 31), u, int(now_lane / 32)); },
                    [&](int u, const Op<T>& k) { mma(k, q[u], s[n]); });
      if (CAP != kNoCap) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = p.from_bend * bend_of<CAP == kFineCap>(s[n][i] * p.to_bend).t;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] *= p.to_log2;
      }
      if (BIAS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x4 at = place[32 * n + 8 * (i / 4) + 4 * half + i % 4];
          const float dx = x - at[0], dy = y - at[1], dz = z - at[2];
          s[n][i] += at[3] - slope * __builtin_amdgcn_sqrtf(dx * dx + dy * dy + dz * dz);
          if (i % 4 == 3) in_turn();
        }
      } else if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] += place[32 * n + 8 * (i / 4) + 4 * half + i % 4][3];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) high = fmaxf(high, s[n][i]);
    }
    high = fmaxf(high, other_half(high));
    if (__any(high > top)) {
      const float now = fmaxf(top, high);
      const float shrink = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - now);
      top = now;
      sum *= shrink;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] *= shrink;
    }
    // a row that has seen no key yet: every exponent is -infinity
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int n = 0; n < KT / 32; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[n][i] = __builtin_amdgcn_exp2f(s[n][i] - base);
        sum += s[n][i];
      }
      Op<T> w[kLineChunks<T>];
#pragma unroll
      for (int c = 0; c < kLineChunks<T>; ++c) register_chunk(s[n], c, w[c]);
      in_flight<kLineChunks<T> * ND>(
          [&](int i) { return column_chunk<DP>(vtile + 32 * n * DP, i / ND, 32 * (i % ND), now_lane); },
          [&](int i, const Op<T>& v) { mma(v, w[i / ND], acc[i % ND]); });
    }
  }
  if (!row.exists) return;
  // Keys are hidden from all rows of a structure or from none.  Scores of hidden keys are
  // -infinity only for rows that are finite themselves: where no key is seen nothing of them counts.
  if (!tiles_of.any) {
    top = -INFINITY;
    sum = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t) acc[t] = zeros();
  }
  sum += other_half(sum);
  const int64_t at = row.token * p.heads + row.head;
  if (SPLIT) {
    const int64_t to = (int64_t(blockIdx.z) * p.queries * p.heads + at);
    store_columns<float, DP>(part + to * p.D, p.D, half, acc, 1.0f);
    if (half == 0) {
      part_stats[2 * to] = top;
      part_stats[2 * to + 1] = sum;
    }
    return;
  }
  // a row that sees no key gives zeros
  store_columns<T, DP>(out + at * p.D, p.D, half, acc, sum == 0.0f ? 0.0f : 1.0f / sum);
  if (log_sums && half == 0) log_sums[at] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Joins the parts of a row, 64 at most: a wave a row; first a lane a part for the parts'
// weights, then a lane a column, eight parts in flight.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(const float* __restrict__ part,
                                                             const float* __restrict__ part_stats, int parts,
                                                             int64_t rows, int D, T* __restrict__ out,
                                                             float* __restrict__ log_sums) {
  constexpr int AHEAD = 8;
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  float top = -INFINITY, sum = 0.0f;
  if (lane < parts) {
    top = part_stats[2 * (lane * rows + row)];
    sum = part_stats[2 * (lane * rows + row) + 1];
  }
  float most = top;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
  float weight = most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - most);
  sum *= weight;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) sum += __shfl_xor(sum, m);
  weight *= sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int c0 = 0; c0 < D; c0 += 64) {
    const int c = c0 + lane;
    float v = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += AHEAD) {
      float x[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        x[k] = k0 + k < parts && c < D ? part[((k0 + k) * rows + row) * D + c] : 0.0f;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) v += __shfl(weight, (k0 + k) & 63) * x[k];
    }
    if (c < D) out[row * D + c] = T(v);
  }
  if (log_sums && lane == 0) log_sums[row] = (most + __builtin_amdgcn_logf(sum)) * kLn2;
}

// The gradients to positions (a sum over heads) and, per workgroup, to slopes.
__global__ __launch_bounds__(256) void attention_force_kernel(const float* __restrict__ row_part,
                                                              const float* __restrict__ key_part, int64_t queries,
                                                              int64_t keys, int heads, int key_heads, bool shared,
                                                              float* __restrict__ positions,
                                                              float* __restrict__ key_positions) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < queries + (shared ? 0 : keys);
       i += int64_t(gridDim.x) * 256) {
    f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool row = i < queries;
    const int64_t k = row ? i : i - queries;
    if (row)
      for (int h = 0; h < heads; ++h) r += *reinterpret_cast<const f32x4*>(row_part + 4 * (k * heads + h));
    if (!row || shared)
      for (int h = 0; h < key_heads; ++h) r += *reinterpret_cast<const f32x4*>(key_part + 4 * (k * key_heads + h));
    float* to = (row ? positions : key_positions) + 3 * k;
    to[0] = r[0];
    to[1] = r[1];
    to[2] = r[2];
  }
}

// dslope_h: a workgroup sums its share of the tokens for one head, a lane a token in turn;
// attention_slope_kernel adds the shares in order.
__global__ __launch_bounds__(256) void attention_slope_part_kernel(const float* __restrict__ row_part, int64_t queries,
                                                                   int heads, float* __restrict__ part) {
  __shared__ float sums[4];
  const int h = blockIdx.y;
  const int64_t each = (queries + gridDim.x - 1) / gridDim.x;
  const int64_t begin = int64_t(blockIdx.x) * each, end = begin + each < queries ? begin + each : queries;
  float s = 0.0f;
  for (int64_t i = begin + threadIdx.x; i < end; i += 256) s += row_part[4 * (i * heads + h) + 3];
#pragma unroll
  for (int m = 1; m < 64; m *= 2) s += __shfl_xor(s, m);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x * int64_t(heads) + h] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}
__global__ __launch_bounds__(64) void attention_slope_kernel(const float* __restrict__ part, int groups, int heads,
                                                             float* __restrict__ slopes) {
  const int h = blockIdx.x;
  float s = 0.0f;
  for (int g = threadIdx.x; g < groups; g += 64) s += part[g * int64_t(heads) + h];
#pragma unroll
  for (int m = 1; m < 64; m *= 2) s += __shfl_xor(s, m);
  if (threadIdx.x == 0) slopes[h] = s;
}

template <typename T, int DP, int NW, bool BIAS, Cap CAP>
int launch_forward(const ForwardPlan& f, const Problem& p, void* out, float* log_sums, void* workspace, hipStream_t s) {
  constexpr int KT = NW > 1 && sizeof(T) == 2 ? 64 : 32;
  float* part = static_cast<float*>(workspace);
  float* stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + f.part_bytes);
  const dim3 grid(unsigned(f.items), unsigned(p.key_heads), unsigned(f.parts));
  if (!fits_grid(f.items, 64 * NW)) return set_error(YE3T_EUNSUPPORTED, "too many rows for one launch");
  if (f.parts == 1) {
    hipLaunchKernelGGL((attention_kernel<T, DP, NW, KT, BIAS, CAP, false>), grid, dim3(64 * NW), 0, s, p,
                       static_cast<T*>(out), log_sums, part, stats);
    return check_launch("attention_kernel");
  }
  hipLaunchKernelGGL((attention_kernel<T, DP, NW, KT, BIAS, CAP, true>), grid, dim3(64 * NW), 0, s, p, static_cast<T*>(out),
                     log_sums, part, stats);
  if (int rc = check_launch("attention_kernel")) return rc;
  const int64_t rows = p.queries * p.heads;
  hipLaunchKernelGGL((attention_join_kernel<T>), dim3(unsigned((rows + 3) / 4)), dim3(256), 0, s, part, stats, f.parts,
                     rows, p.D, static_cast<T*>(out), log_sums);
  return check_launch("attention_join_kernel");
}

struct Forward {
  const ForwardPlan& f;
  const Problem& p;
  void* out;
  float* log_sums;
  void* workspace;
  hipStream_t s;
  template <typename T, int DP, int NW, Cap CAP>
  int capped() const {
    return p.slopes ? launch_forward<T, DP, NW, true, CAP>(f, p, out, log_sums, workspace, s)
                    : launch_forward<T, DP, NW, false, CAP>(f, p, out, log_sums, workspace, s);
  }
  template <typename T, int DP, int NW>
  int waves() const {
    return with_cap<T>(p, [&](auto cap) { return capped<T, DP, NW, decltype(cap)::value>(); });
  }
  template <typename T, int DP>
  int operator()() const {
    return f.waves == 1 ? waves<T, DP, 1>() : waves<T, DP, 4>();
  }
};

}  // namespace
}  // namespace attention
}  // namespace ye3t

using namespace ye3t;
using namespace ye3t::attention;

extern "C" {

int64_t ye3t_hip_atom_attention_workspace_bytes(const ye3t_attention_args* args) {
  clear_error();
  if (!args || check_attention(*args)) return -1;
  return forward_plan(*args).bytes;
}

int ye3t_hip_atom_attention(const ye3t_attention_args* args, void* out, void* log_sums, void* workspace,
                            int64_t workspace_bytes, ye3t_stream_t stream) {
  clear_error();
  YE3T_REQUIRE(args != nullptr, "attention needs arguments");
  if (int rc = check_attention(*args)) return rc;
  if (args->queries == 0) return YE3T_OK;
  if (int rc = check_pointers(*args)) return rc;
  YE3T_REQUIRE(out && args->structures > 0, "attention needs structures and an output");
  const ForwardPlan f = forward_plan(*args);
  YE3T_REQUIRE(f.bytes == 0 || (workspace && workspace_bytes >= f.bytes),
               "the workspace is smaller than ye3t_hip_atom_attention_workspace_bytes");
  const Problem p = problem_of(*args);
  return with_width(args->dtype, p.D, Forward{f, p, out, static_cast<float*>(log_sums), workspace, as_stream(stream)});
}

int64_t ye3t_hip_atom_attention_adjoint_workspace_bytes(const ye3t_attention_args* args, int bias_gradients) {
  clear_error();
  if (!args || check_attention(*args)) return -1;
  return adjoint_plan(*args, bias_gradients != 0).bytes;
}

int ye3t_hip_atom_attention_adjoint(const ye3t_attention_args* args, const void* out, const void* log_sums,
                                    const void* out_adjoint, void* query_adjoint, void* key_adjoint,
                                    void* value_adjoint, void* slopes_adjoint, void* positions_adjoint,
                                    void* key_positions_adjoint, void* workspace, int64_t workspace_bytes,
                                    ye3t_stream_t stream) {
  clear_error();
  YE3T_REQUIRE(args != nullptr, "attention needs arguments");
  if (int rc = check_attention(*args)) return rc;
  if (int rc = check_pointers(*args)) return rc;
  const bool forces = slopes_adjoint != nullptr;
  YE3T_REQUIRE(args->queries == 0 || (out && log_sums && out_adjoint && query_adjoint),
               "the gradient needs the output, its sums, its adjoint and an output for the query's");
  YE3T_REQUIRE(args->keys == 0 || (key_adjoint && value_adjoint), "the gradient needs outputs for key and value");
  YE3T_REQUIRE(!forces || args->slopes, "gradients to slopes and positions need slopes and positions");
  YE3T_REQUIRE(!forces || args->queries == 0 || positions_adjoint, "gradients to slopes and positions come together");
  YE3T_REQUIRE(!forces || !args->key_positions || args->keys == 0 || key_positions_adjoint,
               "key_positions need an output for their gradient");
  const AdjointPlan f = adjoint_plan(*args, forces);
  YE3T_REQUIRE(workspace && workspace_bytes >= f.bytes,
               "the workspace is smaller than ye3t_hip_atom_attention_adjoint_workspace_bytes");
  YE3T_REQUIRE(args->structures > 0 || (args->queries == 0 && args->keys == 0), "attention needs structures");
  const Problem p = problem_of(*args);
  char* work = static_cast<char*>(workspace);
  Gradient g{};
  g.out = out;
  g.adjoint = out_adjoint;
  g.direct = reinterpret_cast<uintptr_t>(out_adjoint) % 16 == 0 &&
             args->head_width % (args->dtype == YE3T_F32 ? kChunk<float> : kChunk<__bf16>) == 0;
  g.log_sums = static_cast<const float*>(log_sums);
  g.along = reinterpret_cast<float*>(work);
  g.dq = query_adjoint;
  g.dk = key_adjoint;
  g.dv = value_adjoint;
  g.row_part = reinterpret_cast<float*>(work + f.along_bytes);
  g.key_part = reinterpret_cast<float*>(work + f.along_bytes + f.row_bytes);
  float* slope_part = reinterpret_cast<float*>(work + f.along_bytes + f.row_bytes + f.key_bytes);
  g.sum_part = reinterpret_cast<float*>(work + f.along_bytes + f.row_bytes + f.key_bytes + f.slope_bytes);
  const hipStream_t s = as_stream(stream);
  if (p.queries > 0)
    if (int rc = launch_row_gradient(args->dtype, f, p, g, forces, s)) return rc;
  if (p.keys > 0)
    if (int rc = launch_key_gradient(args->dtype, f, p, g, forces, s)) return rc;
  if (!forces) return YE3T_OK;
  const bool shared = !args->key_positions && !args->key_offsets;  // keys are the query atoms
  const int64_t atoms = p.queries + (shared ? 0 : p.keys);
  if (atoms > 0) {
    const int64_t groups = (atoms + 255) / 256;
    hipLaunchKernelGGL(attention_force_kernel, dim3(unsigned(groups)), dim3(256), 0, s, g.row_part, g.key_part,
                       p.queries, p.keys, p.heads, p.key_heads, shared, static_cast<float*>(positions_adjoint),
                       static_cast<float*>(key_positions_adjoint));
    if (int rc = check_launch("attention_force_kernel")) return rc;
  }
  hipLaunchKernelGGL(attention_slope_part_kernel, dim3(kSlopeGroups, unsigned(p.heads)), dim3(256), 0, s, g.row_part, p.queries, p.heads,
                     slope_part);
  if (int rc = check_launch("attention_slope_part_kernel")) return rc;
  hipLaunchKernelGGL(attention_slope_kernel, dim3(unsigned(p.heads)), dim3(64), 0, s, slope_part, kSlopeGroups, p.heads,
                     static_cast<float*>(slopes_adjoint));
  return check_launch("attention_slope_kernel");
}

}  // extern "C"
