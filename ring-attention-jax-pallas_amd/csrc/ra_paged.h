// Argument blocks and host launchers of the paged key-value cache: page slots, writes, mean keys, page selection, attention of one
// token per sequence.
#pragma once
#include "ra_common.h"

namespace ra {

constexpr int kMaxRows = RA_MAX_PAGED_ROWS;  // sequences of one call: their prefix sums lie in shared memory
constexpr int kStepKeys = 128;               // keys that a workgroup of the attention kernel takes at a time, 32 a wave
constexpr int kWholeKeys = 1024;             // rows of up to so many keys (by the table) are not shared between workgroups
constexpr int kPagedWorkgroups = 2048, kFewWorkgroups = 512, kStepsEach = 4;
constexpr int kPartRows = 16;                // query heads of a workgroup: the columns of a matrix instruction

struct PageTable {
  const int* at;
  long long sb;
  int width, n_pages, shift;  // page_size = 1 << shift
};

// A pool [page, token, head, dim] of 16-bit elements: strides in elements, `dim` contiguous; offsets within a page fit 32 bits.
struct PoolArg {
  const unsigned short* ptr;
  long long sp;
  int st, sh;
};

struct SlotsArgs {
  int* table;
  long long table_sb;
  int width, B, shift;
  const int *before, *after;
  int* ring;
  int n_pages;
  const int* state;
  long long* slots;
  int n_slots;
  int *starts, *granted, *state_out;
};
hipError_t launch_slots(const SlotsArgs& a, hipStream_t stream);

struct WriteArgs {
  const void *k, *v;
  long long k_st, k_sh, v_st, v_sh;  // of the sources, [token, head, dim]
  PoolArg k_pool, v_pool;
  const long long* slots;
  int T, H, D, shift;
  long long n_slots;  // n_pages * page_size
};
hipError_t launch_write(const WriteArgs& a, int src_dtype, int dtype, hipStream_t stream);

struct MeansArgs {
  PoolArg k;
  PageTable table;
  const int *before, *after;
  unsigned short* means;
  long long means_sp;
  int means_sh, B, H, D;
  int cols;  // chunks of a workgroup (set by the launch)
};
hipError_t launch_means(const MeansArgs& a, int dtype, hipStream_t stream);

struct SelectArgs {
  const unsigned short* q;
  long long q_sb;
  int q_sh;
  const unsigned short* means;
  long long means_sp;
  int means_sh;
  PageTable table;
  const int* lengths;
  int B, H, G, D, count, first, last;
  int heads;  // of a page in one load (set by the launch)
  unsigned long long* keys;  // [B, H, width]
  int* pages;                // [B, H, count]
};
constexpr int kFewPages = 512;  // by the table: so many scores and the choice among them are one kernel's
long long select_workspace(int width, long long rows);
hipError_t launch_select(const SelectArgs& a, int dtype, hipStream_t stream);

struct PagedArgs {
  const unsigned short* q;
  long long q_sb;
  int q_sh;
  PoolArg k, v;
  PageTable table;
  const int* lengths;
  const int* pages;  // [B, H, count]: the pages that are read; NULL: all
  int count;
  int B, H, G, tiles;  // heads of the cache, query heads for each, groups of kPartRows among them
  int window;          // 0: none
  const float* slopes;
  float scale2;        // sm_scale * log2(e)
  unsigned short* out;  // [B, H * G, D]
  float* lse;           // [B, H * G]
  // parts (of the workspace): [2 n_wg, kPartRows, D] and, of each, (maximum, sum); for each (row, head) the first one's place and their number
  float* part;
  float2* stats;
  int2* where;
  int n_wg;
};
struct PagedShape {
  int workgroups;
  bool whole;  // each takes a (row, head) whole
  long long workspace;
};
// For rows of up to `keys` keys and so many (row, head)s.
PagedShape paged_shape(long long keys, long long units, int D);
hipError_t launch_paged(PagedArgs& a, int D, int dtype, const PagedShape& shape, void* workspace, hipStream_t stream);

}  // namespace ra
