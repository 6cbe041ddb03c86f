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
  return sort_plan(rows, species).bytes;
}

int ye3t_hip_species_groups(const void* species_of_rows, int species_bytes, int64_t rows, int64_t species, void* order,
                            void* offsets, void* workspace, int64_t workspace_bytes, ye3t_stream_t stream) {
  clear_error();
  if (int rc = check_species(species_bytes, rows, species)) return rc;
  YE3T_REQUIRE(offsets && (rows == 0 || (species_of_rows && order)), "the groups need the rows' species and two outputs");
  const SortPlan p = sort_plan(rows, species);
  YE3T_REQUIRE(rows == 0 || (workspace && workspace_bytes >= p.bytes),
               "the workspace is smaller than ye3t_hip_species_groups_workspace_bytes");
  const hipStream_t s = as_stream(stream);
  Pair* sorted = nullptr;
  char* work = static_cast<char*>(workspace);
  if (int rc = species_bytes == 4 ? sort_tokens(p, static_cast<const int32_t*>(species_of_rows), rows, species, work, &sorted, s)
                                  : sort_tokens(p, static_cast<const int64_t*>(species_of_rows), rows, species, work, &sorted, s))
    return rc;
  hipLaunchKernelGGL(species_group_kernel, dim3(unsigned(rows / kThreads + 1)), dim3(kThreads), 0, s, sorted, rows,
                     species, static_cast<int32_t*>(order), static_cast<int64_t*>(offsets));
  return check_launch("species_group_kernel");
}

}  // extern "C"
