// Gradient of atom attention, row side.
#include "attention.h"

namespace ye3t {
namespace attention {
namespace {

// Row side: dq, D_i, and the row's part of the gradients to position and slope
// (FORCES).  D_i is the dot product of the output with its adjoint.  With FORCES
// a first walk over the keys sums p, p (go . v) and p |r_i - r_j| instead: D_i
// from the sums does not have a bf16 output's rounding, which would stand out
// in gradients kept in fp32, and with D_i = sum p (go . v) / sum p the dz of a row add
// up to zero as they should, whatever the last bits of the row's log sum are.
// The slope's gradient takes distances from their mean, -sum dz (d - mean d),
// for the same reason.
template <typename T, int DP, int NW, bool BIAS, bool FORCES>
__global__ __launch_bounds__(64 * NW) void attention_row_gradient_kernel(Problem p, Gradient g) {
  constexpr int TILE = 32 * NW, KT = 32, NU = DP / (2 * kChunk<T>), ND = DP / 32;
  __shared__ __align__(16) T ktile[KT * kPitch<T, DP>];
  __shared__ __align__(16) T vtile[KT * kPitch<T, DP>];
  __shared__ f32x4 place[KT];
  const Item item = item_of(p.offsets, p.structures, p.queries, p.group, TILE, blockIdx.x);
  const Span own = span_of(p.offsets, item.structure, p.queries);
  const int64_t rows = int64_t(own.length) * p.group;
  if (item.first < 0 || item.first >= rows) return;
  const Span key = span_of(p.key_offsets, item.structure, p.keys);
  const int key_head = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const Row row = row_of(p, own.begin, item.first + 32 * wave + (lane & 31), rows, key_head);
  const bool busy = item.first + 32 * wave < rows;
  const int64_t at = row.token * p.heads + row.head;

  Op<T> q[NU], go[NU];
  line_operand<T, DP>(row.exists ? static_cast<const T*>(p.q) + row.token * p.q_row + row.head * p.q_head : nullptr,
                      p.D, half, q);
  line_operand<T, DP>(row.exists ? static_cast<const T*>(g.adjoint) + at * p.D : nullptr, p.D, half, go);
  float along = 0.0f;
  if (!FORCES) {
    Op<T> o[NU];
    line_operand<T, DP>(row.exists ? static_cast<const T*>(g.out) + at * p.D : nullptr, p.D, half, o);
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < kChunk<T>; ++e) along += float(o[u][e]) * float(go[u][e]);
    along += other_half(along);
  }
  float x = 0.0f, y = 0.0f, z = 0.0f, slope = 0.0f;
  if (BIAS && row.exists) {
    x = p.positions[3 * row.token];
    y = p.positions[3 * row.token + 1];
    z = p.positions[3 * row.token + 2];
    slope = p.slopes[row.head] * kLog2e;
  }
  // a row that sees no key has the sum 0 and no gradient: p = 0 by `seen`
  const float log_sum = row.exists ? g.log_sums[at] : 0.0f;
  const bool empty = log_sum == -INFINITY;
  const float log_sum2 = empty ? 0.0f : log_sum * kLog2e;

  const int tiles = (key.length + KT - 1) / KT;
  const T* kbase = static_cast<const T*>(p.k) + key_head * p.k_head;
  const T* vbase = static_cast<const T*>(p.v) + key_head * p.v_head;
  Staged<T, DP, KT, 64 * NW> ks, vs;
  f32x4 next_place = {0.0f, 0.0f, 0.0f, 0.0f};
  auto fetch = [&](int t) {
    auto seen = [&](int line) {
      const int j = t * KT + line;
      return j < key.length && (!p.key_mask || p.key_mask[key.begin + j]);
    };
    ks.load(p.D, [&](int line) { return seen(line) ? kbase + (key.begin + t * KT + line) * p.k_row : nullptr; });
    vs.load(p.D, [&](int line) { return seen(line) ? vbase + (key.begin + t * KT + line) * p.v_row : nullptr; });
    if (int(threadIdx.x) < KT) {
      const int j = t * KT + int(threadIdx.x);
      next_place = key_place<BIAS>(p, key.begin + j, j < key.length);
    }
  };
  f32x16 acc[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) acc[t] = zeros();
  float gx = 0.0f, gy = 0.0f, gz = 0.0f, gs = 0.0f, mass = 0.0f, mean = 0.0f;
  for (int walk = FORCES ? 0 : 1; walk < 2; ++walk) {
    if (ks.AHEAD && tiles > 0) fetch(0);
    for (int tile = 0; tile < tiles; ++tile) {
      __syncthreads();
      if (!ks.AHEAD) fetch(tile);
      ks.write(ktile);
      vs.write(vtile);
      if (int(threadIdx.x) < KT) place[threadIdx.x] = next_place;
      __syncthreads();
      if (ks.AHEAD && tile + 1 < tiles) fetch(tile + 1);
      if (!busy) continue;
      f32x16 s = zeros(), dp = zeros();
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        mma(line_chunk<T, DP>(ktile, lane & 31, u, half), q[u], s);
        mma(line_chunk<T, DP>(vtile, lane & 31, u, half), go[u], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const f32x4 k = place[8 * (i / 4) + 4 * half + i % 4];
        float dx = 0.0f, dy = 0.0f, dz = 0.0f, distance = 0.0f;
        if (BIAS) {
          dx = x - k[0], dy = y - k[1], dz = z - k[2];
          distance = __builtin_amdgcn_sqrtf(dx * dx + dy * dy + dz * dz);
        }
        const Weight w = weight_of<BIAS>(p, s[i], log_sum2, slope, distance, k[3] != 0.0f && !empty);
        if (FORCES && walk == 0) {
          along += w.p * dp[i];
          mass += w.p;
          mean += w.p * distance;
          continue;
        }
        const float tilt = w.p * (dp[i] - along);
        s[i] = tilt * w.slant;
        if (FORCES) {
          gs -= tilt * (distance - mean);
          const float pull = distance > 0.0f ? -tilt / distance : 0.0f;
          gx += pull * dx;
          gy += pull * dy;
          gz += pull * dz;
        }
      }
      if (FORCES && walk == 0) continue;
#pragma unroll
      for (int c = 0; c < kLineChunks<T>; ++c) {
        Op<T> w;
        register_chunk(s, c, w);
#pragma unroll
        for (int t = 0; t < ND; ++t) mma(column_chunk<DP>(ktile, c, 32 * t, half), w, acc[t]);
      }
    }
    if (FORCES && walk == 0) {
      mass += other_half(mass);
      const float per = mass > 0.0f ? 1.0f / mass : 0.0f;
      along = (along + other_half(along)) * per;
      mean = (mean + other_half(mean)) * per;
    }
  }
  if (!row.exists) return;
  store_columns<T, DP>(static_cast<T*>(g.dq) + at * p.D, p.D, half, acc, p.scale);
  if (half == 0) g.along[at] = along;
  if (FORCES) {
    const float m = p.slopes[row.head];
    f32x4 r = {gx, gy, gz, gs};
#pragma unroll
    for (int a = 0; a < 4; ++a) r[a] = (r[a] + other_half(r[a])) * (a < 3 ? m : 1.0f);
    if (half == 0) *reinterpret_cast<f32x4*>(g.row_part + 4 * at) = r;
  }
}

template <typename T, int DP, int NW, bool BIAS, bool FORCES>
int launch_rows(const AdjointPlan& f, const Problem& p, const Gradient& g, hipStream_t s) {
  if (!fits_grid(f.row_items, 64 * NW)) return set_error(YE3T_EUNSUPPORTED, "too many rows for one launch");
  hipLaunchKernelGGL((attention_row_gradient_kernel<T, DP, NW, BIAS, FORCES>),
                     dim3(unsigned(f.row_items), unsigned(p.key_heads)), dim3(64 * NW), 0, s, p, g);
  return check_launch("attention_row_gradient_kernel");
}

struct Side {
  const AdjointPlan& f;
  const Problem& p;
  const Gradient& g;
  bool forces;
  hipStream_t s;
  template <typename T, int DP, int NW>
  int waves() const {
    return forces ? launch_rows<T, DP, NW, true, true>(f, p, g, s)
                  : p.slopes ? launch_rows<T, DP, NW, true, false>(f, p, g, s)
                             : launch_rows<T, DP, NW, false, false>(f, p, g, s);
  }
  template <typename T, int DP>
  int operator()() const {
    return f.row_waves == 1 ? waves<T, DP, 1>() : waves<T, DP, 4>();
  }
};

}  // namespace

int launch_row_gradient(int dtype, const AdjointPlan& f, const Problem& p, const Gradient& g, bool forces,
                        hipStream_t s) {
  return with_width(dtype, p.D, Side{f, p, g, forces, s});
}

}  // namespace attention
}  // namespace ye3t
