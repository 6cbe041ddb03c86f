// Stable sorting of positions by token, with no atomics on data: the order depends on
// the tokens alone.
#pragma once

#include "common.h"

namespace ye3t {
namespace {  // kernels of each source that sorts

template <typename Index>
__device__ inline int64_t token_at(const Index* __restrict__ tokens, int64_t i, int64_t vocabulary) {
  const int64_t t = int64_t(tokens[i]);
  return t < 0 || t >= vocabulary ? -1 : t;
}


// ---- sorting ----------------------------------------------------------------
// One pass orders the positions by one digit of their token, stably: every
// workgroup owns an equal run of positions and first counts its digits
// (digit_count_kernel), then places them (digit_place_kernel), starting from
// the counts of lower digits everywhere and of its own digit in the runs before
// it.  Tokens outside the table sort last, as the token `vocabulary`.
constexpr int kBins = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortRuns = 128;

struct Pair {
  uint32_t token, position;
};

// Where sorted positions go: as pairs, or (species.hip) something else.  begin(): the first place of each digit.
struct Pairs {
  Pair* out;
  __device__ inline void put(uint32_t at, const Pair& p) const { out[at] = p; }
  __device__ inline void begin(int, uint32_t) const {}
};

template <bool FIRST, typename Index>
__device__ inline Pair pair_at(const Index* __restrict__ tokens, const Pair* __restrict__ pairs, int64_t i,
                               int64_t vocabulary) {
  if (!FIRST) return pairs[i];
  const int64_t t = token_at(tokens, i, vocabulary);
  return {uint32_t(t < 0 ? vocabulary : t), uint32_t(i)};
}

// The live lanes of the wave that have this lane's digit.
__device__ inline uint64_t lanes_of_digit(uint32_t digit, bool live) {
  uint64_t same = __ballot(live);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1u);
    same &= ((digit >> b) & 1u) ? set : ~set;
  }
  return same;
}

// A digit's counts by wave become the waves' first places; `next` moves past them.
__device__ inline void places_of_waves(uint32_t (*of_wave)[kBins], int digit, uint32_t& next) {
  uint32_t at = next;
#pragma unroll
  for (int w = 0; w < kSortThreads / 64; ++w) {
    const uint32_t n = of_wave[w][digit];
    of_wave[w][digit] = at;
    at += n;
  }
  next = at;
}

template <bool FIRST, typename Index>
__global__ __launch_bounds__(kSortThreads) void digit_count_kernel(const Index* __restrict__ tokens,
                                                                   const Pair* __restrict__ pairs, int64_t N,
                                                                   int64_t run, int64_t vocabulary, int shift,
                                                                   uint32_t* __restrict__ counts) {
  __shared__ uint32_t bins[kBins];
  if (threadIdx.x < kBins) bins[threadIdx.x] = 0;
  __syncthreads();
  const int64_t begin = int64_t(blockIdx.x) * run, end = begin + run < N ? begin + run : N;
  // whole numbers: their sum is the same in any order
  for (int64_t i = begin + threadIdx.x; i < end; i += kSortThreads)
    atomicAdd(&bins[(pair_at<FIRST>(tokens, pairs, i, vocabulary).token >> shift) & (kBins - 1)], 1u);
  __syncthreads();
  if (threadIdx.x < kBins) counts[blockIdx.x * kBins + threadIdx.x] = bins[threadIdx.x];
}

template <bool FIRST, typename Index, typename Out>
__global__ __launch_bounds__(kSortThreads) void digit_place_kernel(const Index* __restrict__ tokens,
                                                                   const Pair* __restrict__ pairs, int64_t N,
                                                                   int64_t run, int64_t vocabulary, int shift,
                                                                   const uint32_t* __restrict__ counts,
                                                                   const Out out) {
  constexpr int kWaves = kSortThreads / 64;
  __shared__ uint32_t next[kBins];            // where this run's next position of a digit goes
  __shared__ uint32_t of_wave[kWaves][kBins];  // a wave's count of a digit, then its place among the waves
  __shared__ uint32_t wave_sums[kBins / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  // The runs' counts of a digit are added by four threads, eight loads of each in flight.
  {
    constexpr int PARTS = kSortThreads / kBins;
    const int digit = t % kBins, part = t / kBins;
    uint32_t before = 0, all = 0;
    for (int r0 = part; r0 < int(gridDim.x); r0 += 8 * PARTS) {
      uint32_t n[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) n[k] = r0 + k * PARTS < int(gridDim.x) ? counts[(r0 + k * PARTS) * kBins + digit] : 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        all += n[k];
        if (r0 + k * PARTS < int(blockIdx.x)) before += n[k];
      }
    }
    of_wave[part][digit] = before;
    of_wave[PARTS + part][digit] = all;
    __syncthreads();
    if (part == 0) {
      before = all = 0;
#pragma unroll
      for (int k = 0; k < PARTS; ++k) before += of_wave[k][digit], all += of_wave[PARTS + k][digit];
      uint32_t sum = all;  // inclusive over the lanes' digits
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const uint32_t up = __shfl_up(sum, m);
        if (lane >= m) sum += up;
      }
      if (lane == 63) wave_sums[wave] = sum;
      next[t] = sum - all + before;
    }
  }
  __syncthreads();
  if (t < kBins)
    for (int w = 0; w < wave; ++w) next[t] += wave_sums[w];
  __syncthreads();
  if (blockIdx.x == 0 && t < kBins) out.begin(t, next[t]);
  const int64_t begin = int64_t(blockIdx.x) * run, end = begin + run < N ? begin + run : N;
  for (int64_t i0 = begin; i0 < end; i0 += kSortThreads) {
    for (int k = t; k < kWaves * kBins; k += kSortThreads) (&of_wave[0][0])[k] = 0;
    __syncthreads();
    const bool live = i0 + t < end;
    const Pair p = live ? pair_at<FIRST>(tokens, pairs, i0 + t, vocabulary) : Pair{0, 0};
    const uint32_t digit = (p.token >> shift) & (kBins - 1);
    const uint64_t same = lanes_of_digit(digit, live);
    const uint32_t rank = uint32_t(__popcll(same & ((uint64_t(1) << lane) - 1)));
    if (live && rank == 0) of_wave[wave][digit] = uint32_t(__popcll(same));
    __syncthreads();
    if (t < kBins) places_of_waves(of_wave, t, next[t]);
    __syncthreads();
    if (live) out.put(of_wave[wave][digit] + rank, p);
    __syncthreads();
  }
}

// All passes over few positions by one workgroup, in LDS: one launch where the
// kernels above take two a pass.  Each wave owns an equal run of positions, counts its digits
// and, once all counts are added up, places them by itself.
constexpr int kSmallSort = 4096;

template <typename Index, typename Out>
__global__ __launch_bounds__(kSortThreads) void small_sort_kernel(const Index* __restrict__ tokens, int N,
                                                                  int64_t vocabulary, int passes,
                                                                  const Out out) {
  constexpr int kWaves = kSortThreads / 64;
  __shared__ Pair held[2][kSmallSort];
  __shared__ uint32_t of_wave[kWaves][kBins];
  __shared__ uint32_t wave_sums[kBins / 64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int run = (N + kSortThreads - 1) / kSortThreads * 64;
  const int begin = wave * run, end = begin + run < N ? begin + run : N;
  for (int i = t; i < N; i += kSortThreads)
    held[0][i] = pair_at<true>(tokens, static_cast<const Pair*>(nullptr), i, vocabulary);
  for (int pass = 0; pass < passes; ++pass) {
    const Pair* in = held[pass & 1];
    Pair* to = held[~pass & 1];
    const int shift = 8 * pass;
    for (int k = t; k < kWaves * kBins; k += kSortThreads) (&of_wave[0][0])[k] = 0;
    __syncthreads();
    for (int i = begin + lane; i < end; i += 64) atomicAdd(&of_wave[wave][(in[i].token >> shift) & (kBins - 1)], 1u);
    __syncthreads();
    uint32_t own = 0, sum = 0;
    if (t < kBins) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) own += of_wave[w][t];
      sum = own;
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const uint32_t up = __shfl_up(sum, m);
        if (lane >= m) sum += up;
      }
      if (lane == 63) wave_sums[wave] = sum;
    }
    __syncthreads();
    if (t < kBins) {
      sum -= own;
      for (int w = 0; w < wave; ++w) sum += wave_sums[w];
      if (pass + 1 == passes) out.begin(t, sum);
      places_of_waves(of_wave, t, sum);
    }
    __syncthreads();
    for (int i0 = begin; i0 < end; i0 += 64) {
      const bool live = i0 + lane < end;
      const Pair p = live ? in[i0 + lane] : Pair{0, 0};
      const uint32_t digit = (p.token >> shift) & (kBins - 1);
      const uint64_t same = lanes_of_digit(digit, live);
      const uint32_t rank = uint32_t(__popcll(same & ((uint64_t(1) << lane) - 1)));
      const uint32_t at = of_wave[wave][digit] + rank;
      __threadfence_block();  // every lane has read its digit's place before it moves on
      if (live && rank == 0) of_wave[wave][digit] = at + uint32_t(__popcll(same));
      __threadfence_block();
      if (live) {
        if (pass + 1 == passes) out.put(at, p);
        else to[at] = p;
      }
    }
    __syncthreads();
  }
}

struct SortPlan {
  int passes;
  int64_t runs, run, pairs_bytes, counts_bytes, bytes;
};

// Runs of at least 2 048 positions, 128 of them at most.
inline SortPlan sort_plan(int64_t N, int64_t vocabulary) {
  SortPlan p{};
  for (p.passes = 1; p.passes < 4 && (vocabulary >> (8 * p.passes)) > 0; ++p.passes) {}
  p.run = (N + kSortRuns - 1) / kSortRuns;
  if (p.run < 2048) p.run = 2048;
  p.runs = (N + p.run - 1) / p.run;
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  p.pairs_bytes = up(N * int64_t(sizeof(Pair)));
  p.counts_bytes = up(p.runs * kBins * 4);
  p.bytes = 2 * p.pairs_bytes + p.counts_bytes;
  return p;
}

template <bool FIRST, typename Index, typename Out>
int sort_pass(const SortPlan& p, const Index* tokens, const Pair* in, int64_t N, int64_t vocabulary, int shift,
              uint32_t* counts, const Out& out, hipStream_t s) {
  hipLaunchKernelGGL((digit_count_kernel<FIRST, Index>), dim3(unsigned(p.runs)), dim3(kSortThreads), 0, s, tokens, in,
                     N, p.run, vocabulary, shift, counts);
  if (int rc = check_launch("digit_count_kernel")) return rc;
  hipLaunchKernelGGL((digit_place_kernel<FIRST, Index, Out>), dim3(unsigned(p.runs)), dim3(kSortThreads), 0, s, tokens,
                     in, N, p.run, vocabulary, shift, counts, out);
  return check_launch("digit_place_kernel");
}

template <typename Index, typename Out>
int small_sort(const SortPlan& p, const Index* tokens, int64_t N, int64_t vocabulary, const Out& out, hipStream_t s) {
  hipLaunchKernelGGL((small_sort_kernel<Index, Out>), dim3(1), dim3(kSortThreads), 0, s, tokens, int(N), vocabulary,
                     p.passes, out);
  return check_launch("small_sort_kernel");
}

// The positions in the order of their tokens, in `p.bytes` of `work`.
template <typename Index>
int sort_tokens(const SortPlan& p, const Index* tokens, int64_t N, int64_t vocabulary, char* work, Pair** sorted,
                hipStream_t s) {
  Pair* pairs[2] = {reinterpret_cast<Pair*>(work), reinterpret_cast<Pair*>(work + p.pairs_bytes)};
  uint32_t* counts = reinterpret_cast<uint32_t*>(work + 2 * p.pairs_bytes);
  *sorted = pairs[(p.passes - 1) & 1];
  if (N > 0 && N <= kSmallSort) return small_sort(p, tokens, N, vocabulary, Pairs{*sorted}, s);
  for (int k = 0; k < p.passes && N > kSmallSort; ++k) {
    const int rc = k == 0 ? sort_pass<true>(p, tokens, static_cast<const Pair*>(nullptr), N, vocabulary, 0, counts, Pairs{pairs[0]}, s)
                          : sort_pass<false>(p, tokens, pairs[(k + 1) & 1], N, vocabulary, 8 * k, counts,
                                            Pairs{pairs[k & 1]}, s);
    if (rc) return rc;
  }
  return YE3T_OK;
}

}  // namespace
}  // namespace ye3t
