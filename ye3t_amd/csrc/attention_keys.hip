// Gradient of atom attention, key side.
#include "attention.h"

namespace ye3t {
namespace attention {
namespace {

// Key side: dk, dv and the key's part of the gradient to its position.  A wave
// owns 32 keys and walks over the rows of its key head in tiles of 32, all heads of
// its group among them, so the sums over shared heads are registers and no atomics
// are needed.
//
// Four products of a tile.  dk and dv take half the registers; with rows of 128 in
// bf16 the keys' v lie in LDS so that two waves fit a SIMD, and where the keys give
// too few workgroups for that the row axis is taken in parts: 8 192 atoms, 16 heads
// of 128 over 4, 1.93 -> 1.48 ms, the matrix units busy for 30 % of the time and the
// vector units for 49 %.  96 structures of 480 atoms with distances and cap, 8 heads of 64:
// 0.32 ms, bound by about 20 vector operations a score.
template <typename T, int DP, int NW, Cap CAP, bool BIAS, bool FORCES>
__global__ __launch_bounds__(64 * NW, (kGradientWaves<T, DP, NW>)) void attention_key_gradient_kernel(Problem p, Gradient g) {
  constexpr int TILE = 32 * NW, RT = 32, NU = DP / (2 * kChunk<T>), ND = DP / 32;
  constexpr int BUFFERS = NW == 1 ? 1 : 2;
  __shared__ __align__(16) T qtiles[BUFFERS * RT * DP];
  __shared__ __align__(16) T gtiles[BUFFERS * RT * DP];
  __shared__ f32x4 places[BUFFERS * RT];  // x, y, z, slope
  __shared__ f32x2 all_stats[BUFFERS * RT];  // log sum, or infinity for a row that sees no key or does not exist; D_i
  constexpr bool KEEP = kKeepLines<T, DP, NW>;
  __shared__ __align__(16) T kept[KEEP ? TILE * DP : 1];
  const Item item = item_of(p.key_offsets, p.structures, p.keys, 1, TILE, blockIdx.x);
  const Span key = span_of(p.key_offsets, item.structure, p.keys);
  if (item.first < 0 || item.first >= key.length) return;
  const Span own = span_of(p.offsets, item.structure, p.queries);
  const int64_t rows = int64_t(own.length) * p.group;
  const int key_head = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int mine = int(item.first) + 32 * wave + (lane & 31);
  const bool exists = mine < key.length;
  const bool busy = int(item.first) + 32 * wave < key.length;
  const int64_t token = key.begin + mine;
  const bool seen = exists && (!p.key_mask || p.key_mask[token]);
  const f32x4 here = key_place<BIAS>(p, token, seen);
  Op<T> k[NU], v[NU];
  line_operand<T, DP>(seen ? static_cast<const T*>(p.k) + token * p.k_row + key_head * p.k_head : nullptr, p.D, half, k);
  line_operand<T, DP>(seen ? static_cast<const T*>(p.v) + token * p.v_row + key_head * p.v_head : nullptr, p.D, half, v);

  T* own_lines = kept + (KEEP ? 32 * wave * DP : 0);
  if constexpr (KEEP) keep_lines<T, DP>(own_lines, v, lane);

  f32x4 next_place = {0.0f, 0.0f, 0.0f, 0.0f};
  f32x2 next_stats = {-INFINITY, 0.0f};
  auto begin = [&](int64_t r0) {
    const int buffer = BUFFERS == 2 ? int(r0 / RT) & 1 : 0;
    load_tile<T, DP, RT, 64 * NW, BUFFERS == 1 || KEEP>(qtiles + buffer * RT * DP, p.D, p.direct, [&](int line) {
      const Row r = row_of(p, own.begin, r0 + line, rows, key_head);
      return r.exists ? static_cast<const T*>(p.q) + r.token * p.q_row + r.head * p.q_head : nullptr;
    });
    load_tile<T, DP, RT, 64 * NW, BUFFERS == 1 || KEEP>(gtiles + buffer * RT * DP, p.D, g.direct, [&](int line) {
      const Row r = row_of(p, own.begin, r0 + line, rows, key_head);
      return r.exists ? static_cast<const T*>(g.adjoint) + (r.token * p.heads + r.head) * p.D : nullptr;
    });
    // nothing here uses what it loads: a wait would be for the tile's rows too
    if (int(threadIdx.x) < RT) {
      const Row r = row_of(p, own.begin, r0 + int(threadIdx.x), rows, key_head);
      next_stats = f32x2{-INFINITY, 0.0f};
      if (r.exists) {
        const int64_t at = r.token * p.heads + r.head;
        next_stats = f32x2{g.log_sums[at], g.along[at]};
        if (BIAS)
          next_place = f32x4{p.positions[3 * r.token], p.positions[3 * r.token + 1], p.positions[3 * r.token + 2],
                             p.slopes[r.head]};
      }
    }
  };
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) dk[t] = dv[t] = zeros();
  float gx = 0.0f, gy = 0.0f, gz = 0.0f;
  // grid axis z: equal parts of the row tiles
  const int64_t each = ((rows + RT - 1) / RT + gridDim.z - 1) / gridDim.z * RT;
  const int64_t start = int64_t(blockIdx.z) * each, until = start + each < rows ? start + each : rows;
  if (BUFFERS == 2 && start < until) begin(start);
  for (int64_t r0 = start; r0 < until; r0 += RT) {
    const int buffer = BUFFERS == 2 ? int(r0 / RT) & 1 : 0;
    if (BUFFERS == 1) {
      __syncthreads();  // the last tile has been used
      begin(r0);
    }
    if (int(threadIdx.x) < RT) {
      const bool counts = next_stats[0] != -INFINITY;
      // A row that sees no key or does not exist: one place for all, with a slope, since zero
      // times the distance of a key too far away is not a number.
      places[buffer * RT + threadIdx.x] =
          counts ? f32x4{next_place[0], next_place[1], next_place[2], next_place[3] * kLog2e} : f32x4{0.0f, 0.0f, 0.0f, 1.0f};
      all_stats[buffer * RT + threadIdx.x] =
          f32x2{counts ? next_stats[0] * kLog2e : INFINITY, counts ? next_stats[1] : 0.0f};
    }
    arrived();
    __syncthreads();
    if (BUFFERS == 2 && r0 + RT < until) begin(r0 + RT);
    const T *qtile = qtiles + buffer * RT * DP, *gtile = gtiles + buffer * RT * DP;
    const f32x4* place = places + buffer * RT;
    const f32x2* stats = all_stats + buffer * RT;
    if (!busy) continue;
    const unsigned now_lane = anew<BUFFERS == 1 || KEEP>(lane) & 63;
    f32x16 s = zeros(), dp = zeros();
    const int own_line = int(now_lane & 31), now_half = int(now_lane / 32);
    if constexpr (KEEP) {
      in_flight<NU, 1>(
          [&](int u) {
            return Three<T>{line_chunk<T, DP>(qtile, own_line, u, now_half), line_chunk<T, DP>(gtile, own_line, u, now_half),
                            line_chunk<T, DP>(own_lines, own_line, u, now_half)};
          },
          [&](int u, const Three<T>& qgv) {
            mma(qgv.a, k[u], s);
            mma(qgv.b, qgv.c, dp);
          });
    } else {
      in_flight<NU>(
          [&](int u) {
            return Two<T>{line_chunk<T, DP>(qtile, own_line, u, now_half), line_chunk<T, DP>(gtile, own_line, u, now_half)};
          },
          [&](int u, const Two<T>& qg) {
            mma(qg.a, k[u], s);
            mma(qg.b, v[u], dp);
          });
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int line = 8 * (i / 4) + 4 * half + i % 4;
      const f32x2 st = stats[line];
      const Score z = score_of<CAP>(p, s[i]);
      float exponent = z.s - st[0], dx = 0.0f, dy = 0.0f, dz = 0.0f, slope = 0.0f, per = 0.0f;
      if (BIAS) {
        const f32x4 r = place[line];
        dx = here[0] - r[0], dy = here[1] - r[1], dz = here[2] - r[2], slope = r[3];
        const float square = dx * dx + dy * dy + dz * dz;
        if (FORCES) {
          per = square >= kLeastSquare ? __builtin_amdgcn_rsqf(fminf(square, kMostSquare)) : 0.0f;
          exponent -= slope * (fminf(square, kMostSquare) * per);
        } else {
          exponent -= slope * __builtin_amdgcn_sqrtf(square);
        }
      }
      const float w = __builtin_amdgcn_exp2f(exponent);
      const float tilt = w * (dp[i] - st[1]);
      s[i] = tilt * z.slant;
      dp[i] = w;
      if (FORCES) {
        const float pull = -tilt * slope * per;
        gx += pull * dx;
        gy += pull * dy;
        gz += pull * dz;
      }
      if (i % 4 == 3) in_turn();
    }
    Op<T> ds[kLineChunks<T>], w[kLineChunks<T>];
#pragma unroll
    for (int c = 0; c < kLineChunks<T>; ++c) {
      register_chunk(s, c, ds[c]);
      register_chunk(dp, c, w[c]);
    }
    in_flight<kLineChunks<T> * ND>(
        [&](int i) {
          return Two<T>{column_chunk<DP>(qtile, i / ND, 32 * (i % ND), now_lane),
                        column_chunk<DP>(gtile, i / ND, 32 * (i % ND), now_lane)};
        },
        [&](int i, const Two<T>& qg) {
          mma(qg.a, ds[i / ND], dk[i % ND]);
          mma(qg.b, w[i / ND], dv[i % ND]);
        });
  }
  if (!exists) return;
  if (!seen) {  // what its scores would have been
    gx = gy = gz = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t) dk[t] = dv[t] = zeros();
  }
  const int64_t at = token * p.key_heads + key_head;
  if (gridDim.z > 1) {
    const int64_t all = p.keys * p.key_heads;
    float* to = g.sum_part + (2 * int64_t(blockIdx.z) * all + at) * p.D;
    store_columns<float, DP>(to, p.D, half, dk, 1.0f);
    store_columns<float, DP>(to + all * p.D, p.D, half, dv, 1.0f);
    return;
  }
  store_columns<T, DP>(static_cast<T*>(g.dk) + at * p.D, p.D, half, dk, p.scale * slant_scale<CAP>());
  store_columns<T, DP>(static_cast<T*>(g.dv) + at * p.D, p.D, half, dv, 1.0f);
  if (FORCES) {
    f32x4 r = {gx, gy, gz, 0.0f};
#pragma unroll
    for (int a = 0; a < 3; ++a) r[a] = (r[a] + other_half(r[a])) * kLn2;  // the slope was in units of log2
    if (half == 0) *reinterpret_cast<f32x4*>(g.key_part + 4 * at) = r;
  }
}

// The parts' sums, a lane a value.
template <typename T>
__global__ __launch_bounds__(256) void attention_key_join_kernel(const float* __restrict__ part, int parts, int64_t count,
                                                                 float scale, T* __restrict__ dk, T* __restrict__ dv) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < 2 * count; i += int64_t(gridDim.x) * 256) {
    float s = 0.0f;
    for (int k = 0; k < parts; ++k) s += part[2 * k * count + i];
    if (i < count) dk[i] = T(s * scale);
    else dv[i - count] = T(s);
  }
}

template <typename T, int DP, int NW, Cap CAP, bool BIAS, bool FORCES>
int launch_keys(const AdjointPlan& f, const Problem& p, const Gradient& g, hipStream_t s) {
  if (!fits_grid(f.key_items, 64 * NW)) return set_error(YE3T_EUNSUPPORTED, "too many keys for one launch");
  hipLaunchKernelGGL((attention_key_gradient_kernel<T, DP, NW, CAP, BIAS, FORCES>),
                     dim3(unsigned(f.key_items), unsigned(p.key_heads), unsigned(f.key_parts)), dim3(64 * NW), 0, s, p, g);
  if (int rc = check_launch("attention_key_gradient_kernel")) return rc;
  if (f.key_parts == 1) return YE3T_OK;
  const int64_t count = p.keys * p.key_heads * p.D, groups = (2 * count + 255) / 256;
  hipLaunchKernelGGL((attention_key_join_kernel<T>), dim3(unsigned(groups < (1 << 20) ? groups : 1 << 20)), dim3(256), 0, s,
                     g.sum_part, f.key_parts, count, p.scale * slant_scale<CAP>(), static_cast<T*>(g.dk),
                     static_cast<T*>(g.dv));
  return check_launch("attention_key_join_kernel");
}

struct Side {
  const AdjointPlan& f;
  const Problem& p;
  const Gradient& g;
  bool forces;
  hipStream_t s;
  template <typename T, int DP, int NW, Cap CAP>
  int capped() const {
    return forces ? launch_keys<T, DP, NW, CAP, true, true>(f, p, g, s)
                  : p.slopes ? launch_keys<T, DP, NW, CAP, true, false>(f, p, g, s)
                             : launch_keys<T, DP, NW, CAP, false, false>(f, p, g, s);
  }
  template <typename T, int DP, int NW>
  int waves() const {
    return with_cap<T>(p, [&](auto cap) { return capped<T, DP, NW, decltype(cap)::value>(); });
  }
  template <typename T, int DP>
  int operator()() const {
    return f.key_waves == 1 ? waves<T, DP, 1>() : waves<T, DP, 4>();
  }
};

}  // namespace

int launch_key_gradient(int dtype, const AdjointPlan& f, const Problem& p, const Gradient& g, bool forces,
                        hipStream_t s) {
  return with_width(dtype, p.D, Side{f, p, g, forces, s});
}

}  // namespace attention
}  // namespace ye3t
