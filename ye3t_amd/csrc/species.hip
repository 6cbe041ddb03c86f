// Atoms grouped by species: a stable order of the rows, and where each species begins.
//
//   order = the rows by species, rows of one species as they came
//   offsets[s] = number of rows of a species below s;  offsets[species]: of all that have one
//
// Rows of no species (outside 0 .. species - 1) come last.  Whole numbers throughout: the
// result is the same in every call.
#include "sort.h"

namespace ye3t {
namespace {

constexpr int kThreads = 256;

// The sort's one pass over up to 255 species writes the order and the offsets by itself: 40 000 rows by two
// launches, 10 us, where pairs and the kernel below took 14.
struct Groups {
  int32_t* order;
  int64_t* offsets;
  int species;
  __device__ inline void put(uint32_t at, const Pair& p) const { order[at] = int32_t(p.position); }
  __device__ inline void begin(int digit, uint32_t at) const {
    if (digit <= species) offsets[digit] = at;
  }
};

// A lane a sorted position, which fills the offsets between its token and the one before it.
__global__ __launch_bounds__(kThreads) void species_group_kernel(const Pair* __restrict__ sorted, int64_t N,
                                                                 int64_t species, int32_t* __restrict__ order,
                                                                 int64_t* __restrict__ offsets) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i > N) return;
  const int64_t from = i == 0 ? 0 : int64_t(sorted[i - 1].token) + 1;
  int64_t to = species;
  if (i < N) {
    const Pair p = sorted[i];
    order[i] = int32_t(p.position);
    to = int64_t(p.token);
  }
  for (int64_t v = from; v <= to; ++v) offsets[v] = i;
}

template <typename Index>
int group(const SortPlan& p, const Index* tokens, int64_t rows, int64_t species, int32_t* order, int64_t* offsets,
          char* work, hipStream_t s) {
  if (rows > 0 && p.passes == 1) {
    const Groups out{order, offsets, int(species)};
    if (rows <= kSmallSort) return small_sort(p, tokens, rows, species, out, s);
    return sort_pass<true>(p, tokens, static_cast<const Pair*>(nullptr), rows, species, 0,
                           reinterpret_cast<uint32_t*>(work), out, s);
  }
  Pair* sorted = nullptr;
  if (int rc = sort_tokens(p, tokens, rows, species, work, &sorted, s)) return rc;
  hipLaunchKernelGGL(species_group_kernel, dim3(unsigned(rows / kThreads + 1)), dim3(kThreads), 0, s, sorted, rows,
                     species, order, offsets);
  return check_launch("species_group_kernel");
}

// Few rows of up to 255 species are sorted in LDS alone.
int64_t workspace_of(int64_t rows, int64_t species) {
  const SortPlan p = sort_plan(rows, species);
  return rows <= kSmallSort && p.passes == 1 ? 0 : p.bytes;
}

int check_species(int bytes, int64_t rows, int64_t species) {
  YE3T_REQUIRE(bytes == 4 || bytes == 8, "species must be int32 or int64");
  YE3T_REQUIRE(rows >= 0 && species >= 0, "row and species counts must not be negative");
  YE3T_REQUIRE(rows < (int64_t(1) << 31) - 256 && species < (int64_t(1) << 24),
               "at most 2^31 - 257 rows and 2^24 - 1 species");
  return YE3T_OK;
}

}  // namespace
}  // namespace ye3t

using namespace ye3t;

extern "C" {

int64_t ye3t_hip_species_groups_workspace_bytes(int64_t rows, int64_t species) {
  clear_error();
  if (check_species(4, rows, species)) return -1;
  return workspace_of(rows, species);
}

int ye3t_hip_species_groups(const void* species_of_rows, int species_bytes, int64_t rows, int64_t species, void* order,
                            void* offsets, void* workspace, int64_t workspace_bytes, ye3t_stream_t stream) {
  clear_error();
  if (int rc = check_species(species_bytes, rows, species)) return rc;
  YE3T_REQUIRE(offsets && (rows == 0 || (species_of_rows && order)), "the groups need the rows' species and two outputs");
  const SortPlan p = sort_plan(rows, species);
  const int64_t bytes = workspace_of(rows, species);
  YE3T_REQUIRE(bytes == 0 || (workspace && workspace_bytes >= bytes),
               "the workspace is smaller than ye3t_hip_species_groups_workspace_bytes");
  const hipStream_t s = as_stream(stream);
  char* work = static_cast<char*>(workspace);
  int32_t* to = static_cast<int32_t*>(order);
  int64_t* ends = static_cast<int64_t*>(offsets);
  return species_bytes == 4 ? group(p, static_cast<const int32_t*>(species_of_rows), rows, species, to, ends, work, s)
                            : group(p, static_cast<const int64_t*>(species_of_rows), rows, species, to, ends, work, s);
}

}  // extern "C"
