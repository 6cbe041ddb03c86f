// Gradient of atom attention, row side.
#include "attention.h"

namespace ye3t {
namespace attention {
namespace {

// Row side: dq, D_i, and the row's part of the gradients to position and slope
// (FORCES).
//
// D_i starts as the dot product of the output with its adjoint.  A bf16 output's
// rounding would stand out: it shifts all dz_ij of a row by p_ij times the same
// amount, up to 2^-8 of the largest terms where few keys carry the row.  The dz
// of a row add up to zero, so what they add up to instead is that amount c (the p
// of a row add up to 1 to within fp32's rounding).  Everything here is linear in
// it and is set right after the walk over the keys, dq by the product of the p (and
// the slants) with the keys.  The key side starts from the D_i that is right.
// fp32 calls have no such rounding in dq, and correct only what FORCES sums, where
// terms of many keys cancel.
//
// A row whose log sum is -infinity sees no key.  Its scores are -infinity only where the
// row itself is finite, so its sums are cleared.
//
// Four products of a tile in bf16 (scores, go . v, dq, the p times the keys),
// three in fp32.  dq and its correction take half the registers; with rows of 128
// in bf16 the go lie in LDS so that two waves fit a SIMD: 8 192 atoms, 16 heads of
// 128 over 4, 1.78 -> 1.25 ms, the matrix units busy for 37 % of the time and the vector
// units for 56 %.  96 structures of 480 atoms with distances and cap, 8 heads of 64: 0.32 ms,
// bound by about 25 vector operations a score.
template <typename T, int DP, int NW, Cap CAP, bool BIAS, bool FORCES>
__global__ __launch_bounds__(64 * NW, (kGradientWaves<T, DP, NW>)) void attention_row_gradient_kernel(Problem p, Gradient g) {
  constexpr int TILE = 32 * NW, KT = 32, NU = DP / (2 * kChunk<T>), ND = DP / 32;
  constexpr int BUFFERS = NW == 1 ? 1 : 2;
  __shared__ __align__(16) T ktiles[BUFFERS * KT * DP];
  __shared__ __align__(16) T vtiles[BUFFERS * KT * DP];
  __shared__ f32x4 places[BUFFERS * KT];
  constexpr bool KEEP = kKeepLines<T, DP, NW>;
  __shared__ __align__(16) T kept[KEEP ? TILE * DP : 1];
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
  {
    Op<T> o[NU];
    line_operand<T, DP>(row.exists ? static_cast<const T*>(g.out) + at * p.D : nullptr, p.D, half, o);
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < kChunk<T>; ++e) along += float(o[u][e]) * float(go[u][e]);
    along += other_half(along);
  }
  T* own_lines = kept + (KEEP ? 32 * wave * DP : 0);
  if constexpr (KEEP) keep_lines<T, DP>(own_lines, go, lane);
  float x = 0.0f, y = 0.0f, z0 = 0.0f, slope = 0.0f;
  if (BIAS && row.exists) {
    x = p.positions[3 * row.token];
    y = p.positions[3 * row.token + 1];
    z0 = p.positions[3 * row.token + 2];
    slope = p.slopes[row.head] * kLog2e;
  }
  const float log_sum = row.exists ? g.log_sums[at] : -INFINITY;
  const float log_sum2 = log_sum == -INFINITY ? INFINITY : log_sum * kLog2e;

  const int tiles = (key.length + KT - 1) / KT;
  KeyTiles<T, DP, KT, 64 * NW, BUFFERS, BUFFERS == 1 || KEEP, BIAS> tiles_of{
      p,      key,    static_cast<const T*>(p.k) + key_head * p.k_head, static_cast<const T*>(p.v) + key_head * p.v_head,
      ktiles, vtiles, places};
  constexpr bool RIGHT = sizeof(T) == 2;  // dq is set right
  f32x16 acc[ND], own_keys[RIGHT ? ND : 1];
#pragma unroll
  for (int t = 0; t < ND; ++t) acc[t] = zeros();
#pragma unroll
  for (int t = 0; t < (RIGHT ? ND : 1); ++t) own_keys[t] = zeros();
  // Sums over the keys of dz, and with FORCES of dz and p times the distance and
  // the direction.  Each tile's are summed by themselves first:
  // long sums whose terms cancel keep a few more bits.
  struct Sums {
    float dz, far_dz, far_p;
    f32x4 to_dz, to_p;
    __device__ inline void add(const Sums& o) {
      dz += o.dz, far_dz += o.far_dz, far_p += o.far_p, to_dz += o.to_dz, to_p += o.to_p;
    }
  };
  const Sums none = {0.0f, 0.0f, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
  Sums all = none;
  if (tiles > 0) tiles_of.start(0);
  for (int tile = 0; tile < tiles; ++tile) {
    tiles_of.take(tile, tiles);
    const T *ktile = tiles_of.keys(tile), *vtile = tiles_of.values(tile);
    const f32x4* place = tiles_of.places_of(tile);
    if (!busy) continue;
    const unsigned now_lane = anew<BUFFERS == 1 || KEEP>(lane) & 63;
    f32x16 s = zeros(), dp = zeros();
    const int line = int(now_lane & 31), now_half = int(now_lane / 32);
    if constexpr (KEEP) {
      in_flight<NU, 1>(
          [&](int u) {
            return Three<T>{line_chunk<T, DP>(ktile, line, u, now_half), line_chunk<T, DP>(vtile, line, u, now_half),
                            line_chunk<T, DP>(own_lines, line, u, now_half)};
          },
          [&](int u, const Three<T>& kvg) {
            mma(kvg.a, q[u], s);
            mma(kvg.b, kvg.c, dp);
          });
    } else {
      in_flight<NU>(
          [&](int u) {
            return Two<T>{line_chunk<T, DP>(ktile, line, u, now_half), line_chunk<T, DP>(vtile, line, u, now_half)};
          },
          [&](int u, const Two<T>& kv) {
            mma(kv.a, q[u], s);
            mma(kv.b, go[u], dp);
          });
    }
    Sums now = none;
    const bool masked = p.key_mask != nullptr || (tile + 1) * KT > key.length;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const Score z = score_of<CAP>(p, s[i]);
      float exponent = z.s - log_sum2, dx = 0.0f, dy = 0.0f, dz = 0.0f, distance = 0.0f, per = 0.0f;
      if (BIAS) {
        const f32x4 k = place[8 * (i / 4) + 4 * half + i % 4];
        dx = x - k[0], dy = y - k[1], dz = z0 - k[2];
        const float square = dx * dx + dy * dy + dz * dz;
        if (FORCES) {
          per = square >= kLeastSquare ? __builtin_amdgcn_rsqf(fminf(square, kMostSquare)) : 0.0f;
          distance = fminf(square, kMostSquare) * per;
        } else {
          distance = __builtin_amdgcn_sqrtf(square);
        }
        exponent += k[3] - slope * distance;
      } else if (masked) {
        exponent += place[8 * (i / 4) + 4 * half + i % 4][3];
      }
      const float w = __builtin_amdgcn_exp2f(exponent);
      const float tilt = w * (dp[i] - along);
      s[i] = tilt * z.slant;
      if (RIGHT) dp[i] = w * z.slant;
      if (RIGHT || FORCES) now.dz += tilt;
      if (FORCES) {
        now.far_dz += tilt * distance;
        now.far_p += w * distance;
        const float a = tilt * per, b = w * per;
        now.to_dz[0] += a * dx, now.to_dz[1] += a * dy, now.to_dz[2] += a * dz;
        now.to_p[0] += b * dx, now.to_p[1] += b * dy, now.to_p[2] += b * dz;
      }
      if (i % 4 == 3) in_turn();
    }
    all.add(now);
    Op<T> w[kLineChunks<T>], m[RIGHT ? kLineChunks<T> : 1];
#pragma unroll
    for (int c = 0; c < kLineChunks<T>; ++c) {
      register_chunk(s, c, w[c]);
      if constexpr (RIGHT) register_chunk(dp, c, m[c]);
    }
    in_flight<kLineChunks<T> * ND>([&](int i) { return column_chunk<DP>(ktile, i / ND, 32 * (i % ND), now_lane); },
                                   [&](int i, const Op<T>& k) {
                                     mma(k, w[i / ND], acc[i % ND]);
                                     if constexpr (RIGHT) mma(k, m[i / ND], own_keys[i % ND]);
                                   });
  }
  float off = RIGHT || FORCES ? all.dz + other_half(all.dz) : 0.0f;
  along += off;
  if (!row.exists) return;
  if (log_sum == -INFINITY) {  // a row that sees no key has no gradient, whatever it holds
    off = along = 0.0f;
    all = none;
#pragma unroll
    for (int t = 0; t < ND; ++t) acc[t] = zeros();
#pragma unroll
    for (int t = 0; t < (RIGHT ? ND : 1); ++t) own_keys[t] = zeros();
  }
  if (RIGHT) {
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][i] -= off * own_keys[t][i];
  }
  store_columns<T, DP>(static_cast<T*>(g.dq) + at * p.D, p.D, half, acc, p.scale * slant_scale<CAP>());
  if (half == 0) g.along[at] = along;
  if (FORCES) {
    const float m = p.slopes[row.head];
    f32x4 r;
#pragma unroll
    for (int a = 0; a < 3; ++a) r[a] = -m * ((all.to_dz[a] + other_half(all.to_dz[a])) - off * (all.to_p[a] + other_half(all.to_p[a])));
    r[3] = -((all.far_dz + other_half(all.far_dz)) - off * (all.far_p + other_half(all.far_p)));
    if (half == 0) *reinterpret_cast<f32x4*>(g.row_part + 4 * at) = r;
  }
}

template <typename T, int DP, int NW, Cap CAP, bool BIAS, bool FORCES>
int launch_rows(const AdjointPlan& f, const Problem& p, const Gradient& g, hipStream_t s) {
  if (!fits_grid(f.row_items, 64 * NW)) return set_error(YE3T_EUNSUPPORTED, "too many rows for one launch");
  hipLaunchKernelGGL((attention_row_gradient_kernel<T, DP, NW, CAP, BIAS, FORCES>),
                     dim3(unsigned(f.row_items), unsigned(p.key_heads)), dim3(64 * NW), 0, s, p, g);
  return check_launch("attention_row_gradient_kernel");
}

struct Side {
  const AdjointPlan& f;
  const Problem& p;
  const Gradient& g;
  bool forces;
  hipStream_t s;
  template <typename T, int DP, int NW, Cap CAP>
  int capped() const {
    return forces ? launch_rows<T, DP, NW, CAP, true, true>(f, p, g, s)
                  : p.slopes ? launch_rows<T, DP, NW, CAP, true, false>(f, p, g, s)
                             : launch_rows<T, DP, NW, CAP, false, false>(f, p, g, s);
  }
  template <typename T, int DP, int NW>
  int waves() const {
    return with_cap<T>(p, [&](auto cap) { return capped<T, DP, NW, decltype(cap)::value>(); });
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
