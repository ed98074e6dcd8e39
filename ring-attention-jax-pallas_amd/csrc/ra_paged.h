// Argument blocks and host launchers of the paged key-value cache: page slots, writes, mean keys, page selection, attention of one
// token per sequence.
#pragma once
#include "ra_common.h"

namespace ra {

constexpr int kStepKeys = 128;               // keys that a workgroup of the attention kernel takes at a time, 32 a wave
// A (row, head) is one workgroup's where its keys and values by the table are at most 256 KB (keys x D up to kWholeSize), which a compute unit
// reads in some 6 us, or up to kWholeKeys keys where there are kWholeUnits of them; else the call's keys are shared between workgroups and their parts
// joined, for 4 us and a launch more.  Whole | shared in a graph, us: 512 keys, D=128, 8 (row, head)s 7.2 | 8.8, 128 of them 10.8 | 13.5, 1024 48.7 | 47.9;
// 1024 keys, D=128, 8: 10.4 | 9.1, 32: 12.4 | 10.3, 128: 16.1 | 18.5, 256: 27.9 | 28.2, 1024: 99.6 | 92.2; 2048 keys, D=128, 8: 17.8 | 9.4, 128: 34.5 | 29.0;
// 1000 keys, D=64, 8: 8.4 | 7.5 (from the host, which launches one kernel instead of two, 8.1 | 11), 128: 10.4 | 14.5, 1024: 45.3 | 61.3.
// (The crossing goes by the number of keys more than by their bytes: 1000 keys of D=64 are taken whole for the host's sake, and lose 0.9 us in a graph.)  Lengths are not known
// here: short rows in a table made for longer ones are shared.  1000 keys of 8 heads, D=64, by a table of 63 pages | of 1024 to 8192: in a graph 8.7 | 7.7, from the host 9.0 | 10.5.
constexpr int kWholeSize = 65536, kWholeKeys = 1024, kWholeUnits = 128;
// Workgroups that share: kStepsEach steps for each (128 keys), and at least kFewWorkgroups, two on each compute unit as their registers allow at D = 128 (three, with registers spilled: 391 us for 335; at D = 96, 64 and 32 three, four and five fit, which
// the rule does not use: its figures are D = 128's); at most
// kPagedWorkgroups, whose ends a large call does not feel.  2.15 GB: 1024 workgroups 354 us, 2048 335, 4096 329, but 2.06 GB of 64 rows 336
// with 2048 and 344 with 4096; 231 MB: 2 steps each 49.2, 4: 48.5, 8: 50.6; at least 256 workgroups instead of 512: 20 MB 14.6 instead of 13.7, 768: 134 MB
// 54.1 instead of 50.4.
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

// n floats of host memory to the device in the order of the stream, as kernel arguments.
hipError_t launch_put(const float* values, int n, float* to, hipStream_t stream);

}  // namespace ra
