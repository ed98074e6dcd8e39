// A key-value cache in pages: which page holds which token (slots), writing into pages, the mean keys of pages, the choice of pages by
// those, and attention of one token per sequence over its pages.
#include "ra_paged.h"

namespace ra {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2), aligned(4))) unsigned int u32x2a;
typedef __attribute__((ext_vector_type(3), aligned(4))) unsigned int u32x3a;

struct BF16 {
  static RA_DEV float up(unsigned short x) { return __uint_as_float((unsigned)x << 16); }
  static RA_DEV unsigned down2(float lo, float hi) { return __builtin_bit_cast(unsigned, (bf16x2){(bf16_t)lo, (bf16_t)hi}); }
  static RA_DEV f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static constexpr float kLift = 0.f;
  static RA_DEV unsigned cut2(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }
  static RA_DEV float rest(float w, float lack) { return __builtin_fmaf(w, 0x1p-31f, lack); }
};
struct F16 {
  static RA_DEV float up(unsigned short x) { return (float)__builtin_bit_cast(_Float16, x); }
  static RA_DEV unsigned down2(float lo, float hi) { return __builtin_bit_cast(unsigned, (f16x2){(_Float16)lo, (_Float16)hi}); }
  static RA_DEV f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  // Weights go into the matrix unit as 2^15 times their value: 2^17 of them that are 2^-25 of the largest, each below fp16's least, make up 2^-8 of
  // the output.
  static constexpr float kLift = 15.f;
  static RA_DEV unsigned cut2(float lo, float hi) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(lo, hi)); }
  static RA_DEV float rest(float, float lack) { return fmaxf(lack, 0x1p-24f); }
};

RA_DEV int pages_of(int tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }

// A lane's value from the lanes before it, `id` where there is none: 1, 2, 4, 8 lanes back within a row of sixteen, then the last lane of the row
// and of the half before.  These moves are part of an addition; a shuffle goes through shared memory, ten times as long.
template <int CTRL, int ROWS = 0xf>
RA_DEV int lane_before(int id, int x) { return __builtin_amdgcn_update_dpp(id, x, CTRL, ROWS, 0xf, false); }
RA_DEV int scan_sum(int x) {
  x += lane_before<0x111>(0, x);
  x += lane_before<0x112>(0, x);
  x += lane_before<0x114>(0, x);
  x += lane_before<0x118>(0, x);
  x += lane_before<0x142, 0xa>(0, x);
  x += lane_before<0x143, 0xc>(0, x);
  return x;
}
template <int CTRL, int ROWS = 0xf>
RA_DEV float float_before(float id, float x) { return __int_as_float(lane_before<CTRL, ROWS>(__float_as_int(id), __float_as_int(x))); }
RA_DEV float last_lane(float x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63)); }
RA_DEV float sum_of_wave(float x) {
  x += float_before<0x111>(0.f, x);
  x += float_before<0x112>(0.f, x);
  x += float_before<0x114>(0.f, x);
  x += float_before<0x118>(0.f, x);
  x += float_before<0x142, 0xa>(0.f, x);
  x += float_before<0x143, 0xc>(0.f, x);
  return last_lane(x);
}
RA_DEV float max_of_wave(float x) {
  x = fmaxf(x, float_before<0x111>(RA_NEG_INF, x));
  x = fmaxf(x, float_before<0x112>(RA_NEG_INF, x));
  x = fmaxf(x, float_before<0x114>(RA_NEG_INF, x));
  x = fmaxf(x, float_before<0x118>(RA_NEG_INF, x));
  x = fmaxf(x, float_before<0x142, 0xa>(RA_NEG_INF, x));
  x = fmaxf(x, float_before<0x143, 0xc>(RA_NEG_INF, x));
  return last_lane(x);
}
// ... of the four lanes l, l ^ 16, l ^ 32, l ^ 48, in each of them.
RA_DEV float max_of_rows(float x) {
  const unsigned u = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
RA_DEV float sum_of_rows(float x) {
  const unsigned u = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Sums of numbers >= 0 that stop at 2^31 - 1: the order of additions does not change what they are.
RA_DEV int capped_sum(int x, int y) { return (int)min((unsigned)x + (unsigned)y, 0x7fffffffu); }
RA_DEV int scan_capped(int x) {
  x = capped_sum(x, lane_before<0x111>(0, x));
  x = capped_sum(x, lane_before<0x112>(0, x));
  x = capped_sum(x, lane_before<0x114>(0, x));
  x = capped_sum(x, lane_before<0x118>(0, x));
  x = capped_sum(x, lane_before<0x142, 0xa>(0, x));
  x = capped_sum(x, lane_before<0x143, 0xc>(0, x));
  return x;
}

// Exclusive prefix sums of N values >= 0 of each row, sums[n][0 .. B] in shared memory, so that whatever walks the rows' items in one line finds an
// item's row by halving; all NT threads, neighbouring rows in a thread.  `values(row, x)` is called twice where B > NT.  CAPPED: the first
// value's sums may pass 2^31 - 1, and stop there.
template <int NT, int N, bool CAPPED = false, class F>
RA_DEV void scan_rows(int B, F values, int* const (&sums)[N], int (&red)[NT / 64][N]) {
  auto plus = [](int n, int x, int y) { return CAPPED && n == 0 ? capped_sum(x, y) : x + y; };
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (B + NT - 1) / NT, from = threadIdx.x * per, to = min(from + per, B);
  int x[N], mine[N], s[N];
#pragma unroll
  for (int n = 0; n < N; ++n) mine[n] = 0;
  for (int i = from; i < to; ++i) {
    values(i, x);
#pragma unroll
    for (int n = 0; n < N; ++n) mine[n] = plus(n, mine[n], x[n]);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    // (a sum that has stopped does not say what it was without this lane's value: that of the lane before does)
    const bool capped = CAPPED && n == 0;
    const int upto = capped ? scan_capped(mine[n]) : scan_sum(mine[n]);
    if (lane == 63) red[wave][n] = upto;
    s[n] = capped ? __shfl_up(upto, 1, 64) : upto - mine[n];
    if (capped && lane == 0) s[n] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      s[n] = plus(n, s[n], w < wave ? red[w][n] : 0);
      all = plus(n, all, red[w][n]);
    }
    if (threadIdx.x == 0) sums[n][B] = all;
  }
  for (int i = from; i < to; ++i) {
#pragma unroll
    for (int n = 0; n < N; ++n) sums[n][i] = s[n];
    if (per == 1) break;
    values(i, x);
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = plus(n, s[n], x[n]);
  }
  __syncthreads();
}
// The row that item i < sums[B] belongs to: the last one whose sum is <= i.
RA_DEV int row_of(const int* sums, int B, int i) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---------------------------------------------------------------------------------------
// slots
// ---------------------------------------------------------------------------------------
// Row b goes from before[b] to after[b] tokens.  Pages are taken from the head of the ring of free pages and given back behind its end, both in the
// order of the rows, so every place follows from prefix sums over the rows: each workgroup makes those for itself, and no workgroup waits for
// another.  What is read (the ring's free part, the rows that end) is never what is written (the part behind it, the rows
// that grow).  Latency bound: lengths, sums, a row's page, the slot.  A step of 8 sequences 2.8 us, of 512 with 40500 new tokens 6.1 (a thread each,
// up to 512 workgroups: two tokens a thread one after another took 7.5); an empty kernel's time is 2.3.
constexpr int kSlotThreads = 256;
__global__ __launch_bounds__(kSlotThreads) void slots_kernel(const SlotsArgs a) {
  extern __shared__ int s_mem[];
  __shared__ int red[kSlotThreads / 64][3];
  int* s_new = s_mem;
  int* s_take = s_new + a.B + 1;
  int* s_give = s_take + a.B + 1;
  const int size = 1 << a.shift, cap = a.width << a.shift, tid = threadIdx.x;
  const int P = a.n_pages;
  const int first = (int)((unsigned)max(a.state[0], 0) % (unsigned)P), count = min(max(a.state[1], 0), P);
  auto old_of = [&](int b) { return min(max(a.before[b], 0), cap); };
  auto had_of = [&](int b) { return pages_of(old_of(b), a.shift); };
  auto wants_of = [&](int b) { return pages_of(min(max(a.after[b], 0), cap), a.shift); };
  // (pages fit 31 bits in all, as the table's entries do; tokens that are asked for need not)
  scan_rows<kSlotThreads, 3, true>(
      a.B,
      [&](int b, int (&x)[3]) {
        const int n = a.before[b], m = a.after[b];
        const int pages = pages_of(min(max(m, 0), cap), a.shift) - pages_of(min(max(n, 0), cap), a.shift);
        x[0] = max(max(m, 0) - max(n, 0), 0);
        x[1] = max(pages, 0);
        x[2] = max(-pages, 0);
      },
      {s_new, s_take, s_give}, red);
  const int take = s_take[a.B], give = s_give[a.B];
  // what row b holds from now on: no more than its pages do
  auto granted_of = [&](int b) {
    const int n = old_of(b), m = min(max(a.after[b], 0), cap);
    if (m <= n) return m;
    const int got = min(s_take[b + 1] - s_take[b], max(count - s_take[b], 0));
    return min(m, (pages_of(n, a.shift) + got) << a.shift);
  };
  // (unsigned: a step behind the last of 2^31 - 1 is one, too)
  const unsigned stride = gridDim.x * kSlotThreads, me = blockIdx.x * kSlotThreads + tid;
  for (int b = (int)me; b < a.B; b += (int)stride) {
    a.granted[b] = granted_of(b);
    a.starts[b] = s_new[b];
  }
  if (me == 0) {
    const int used = min(take, count);
    a.starts[a.B] = s_new[a.B];
    a.state_out[0] = (int)(((unsigned)first + (unsigned)used) % (unsigned)P);
    a.state_out[1] = (int)min((unsigned)(count - used) + (unsigned)give, (unsigned)P);
  }
  auto ring_at = [&](int r) { return (int)(((unsigned)first + (unsigned)r) % (unsigned)P); };
  for (unsigned t = me; t < (unsigned)a.n_slots; t += stride) {
    long long slot = -1;
    if ((int)t < s_new[a.B]) {
      const int b = row_of(s_new, a.B, (int)t), n = old_of(b), position = n + ((int)t - s_new[b]);
      if (position >= n && position < granted_of(b)) {
        const int j = position >> a.shift, had = pages_of(n, a.shift);
        const int page = j < had ? a.table[b * a.table_sb + j] : a.ring[ring_at(s_take[b] + j - had)];
        if (page >= 0 && page < P) slot = (long long)page * size + (position & (size - 1));
      }
    }
    a.slots[t] = slot;
  }
  // (the rest from other workgroups on: the first one has had the rows)
  auto from = [&](unsigned third) { return (blockIdx.x + gridDim.x * third / 3) % gridDim.x * kSlotThreads + tid; };
  for (unsigned i = from(1); i < (unsigned)min(take, count); i += stride) {
    const int b = row_of(s_take, a.B, (int)i);
    a.table[b * a.table_sb + had_of(b) + ((int)i - s_take[b])] = a.ring[ring_at((int)i)];
  }
  for (unsigned i = from(2); i < (unsigned)give; i += stride) {
    const int b = row_of(s_give, a.B, (int)i);
    a.ring[(int)(((unsigned)ring_at(count) + i) % (unsigned)P)] = a.table[b * a.table_sb + wants_of(b) + ((int)i - s_give[b])];
  }
}

hipError_t launch_slots(const SlotsArgs& a, hipStream_t stream) {
  // (items: up to 2^31 - 1)
  const int items = a.n_slots > a.B ? a.n_slots : a.B, wgs = (items - 1) / kSlotThreads + 1;
  hipLaunchKernelGGL(slots_kernel, dim3(wgs < 512 ? wgs : 512), dim3(kSlotThreads), 3 * (a.B + 1) * sizeof(int), stream, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// writes
// ---------------------------------------------------------------------------------------
// Eight elements of a token's key and of its value per thread, neighbouring threads on neighbouring chunks.  HBM bound: 30005 tokens of 8 x 96
// from 32 bits to fp16, 277 MB, 49 us (5.7 TB/s); 64 tokens of 8 x 128 2.5.
template <class S, class T>
RA_DEV u32x4 load8(const void* base, long long at) {
  if constexpr (__is_same(S, float)) {
    const f32x4 x = *(const f32x4*)((const float*)base + at), y = *(const f32x4*)((const float*)base + at + 4);
    return (u32x4){T::down2(x[0], x[1]), T::down2(x[2], x[3]), T::down2(y[0], y[1]), T::down2(y[2], y[3])};
  } else {
    const u32x4 x = *(const u32x4*)((const unsigned short*)base + at);
    if constexpr (__is_same(S, T)) return x;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = T::down2(S::up((unsigned short)x[i]), S::up((unsigned short)(x[i] >> 16)));
    return r;
  }
}
template <class S, class T>
__global__ __launch_bounds__(256) void write_kernel(const WriteArgs a) {
  const unsigned cpr = (unsigned)a.D / 8, line = cpr * (unsigned)a.H;
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  const long long t = i / line;
  if (t >= a.T) return;
  const long long slot = a.slots[t];
  if (slot < 0 || slot >= a.n_slots) return;
  const unsigned in_line = i - (unsigned)t * line, h = in_line / cpr, d = 8 * (in_line - h * cpr);
  const long long page = slot >> a.shift;
  const int off = (int)(slot & ((1 << a.shift) - 1));
  const u32x4 k = load8<S, T>(a.k, t * a.k_st + h * a.k_sh + d), v = load8<S, T>(a.v, t * a.v_st + h * a.v_sh + d);
  *(u32x4*)const_cast<unsigned short*>(a.k_pool.ptr + page * a.k_pool.sp + (off * a.k_pool.st + (int)h * a.k_pool.sh + (int)d)) = k;
  *(u32x4*)const_cast<unsigned short*>(a.v_pool.ptr + page * a.v_pool.sp + (off * a.v_pool.st + (int)h * a.v_pool.sh + (int)d)) = v;
}

hipError_t launch_write(const WriteArgs& a, int src_dtype, int dtype, hipStream_t stream) {
  const long long chunks = (long long)a.T * a.H * (a.D / 8);
  const dim3 grid((unsigned)((chunks + 255) / 256));
  const bool half = dtype == RA_DTYPE_F16;
  void (*kernel)(WriteArgs) = half ? write_kernel<BF16, F16> : write_kernel<BF16, BF16>;
  if (src_dtype == RA_DTYPE_F32) kernel = half ? write_kernel<float, F16> : write_kernel<float, BF16>;
  else if (src_dtype == RA_DTYPE_F16) kernel = half ? write_kernel<F16, F16> : write_kernel<F16, BF16>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// mean keys
// ---------------------------------------------------------------------------------------
// The mean over the tokens that a page holds, for each page whose tokens change between before[b] and after[b]: a workgroup per page and up to 64 chunks
// of eight elements, its threads on neighbouring chunks and, beyond those, on different tokens.  HBM bound for prompts (46 MB, 12.3 us), latency for a
// step (64 pages of 8 x 128: 4.8 us of lengths, sums, a page, its keys, the sum over threads).
constexpr int kMeanThreads = 256;
template <class T>
__global__ __launch_bounds__(kMeanThreads) void means_kernel(const MeansArgs a) {
  extern __shared__ int s_first[];
  __shared__ int red[kMeanThreads / 64][1];
  __shared__ float s_sum[kMeanThreads][9];  // (nine words apart: no two of a wave's rows in one bank)
  const int size = 1 << a.table.shift, cap = a.table.width << a.table.shift, tid = threadIdx.x;
  auto low = [&](int b) { return min(max(min(a.before[b], a.after[b]), 0), cap) >> a.table.shift; };
  scan_rows<kMeanThreads, 1>(
      a.B,
      [&](int b, int (&x)[1]) {
        x[0] = a.before[b] == a.after[b] ? 0 : max(pages_of(min(max(a.after[b], 0), cap), a.table.shift) - low(b), 0);
      },
      {s_first}, red);
  const int total = s_first[a.B];
  const int cpr = a.D / 8, line = cpr * a.H, cols = a.cols;
  const int chunk = blockIdx.y * cols + tid % cols, step = kMeanThreads / cols, r0 = tid / cols;
  const int h = chunk / cpr, d = 8 * (chunk % cpr);
  for (unsigned next = blockIdx.x; next < (unsigned)total; next += gridDim.x) {  // (of up to 2^31 - 1: a step behind them is no int)
    const int i = (int)next, b = row_of(s_first, a.B, i), j = low(b) + (i - s_first[b]);
    const int n = min(size, min(max(a.after[b], 0), cap) - (j << a.table.shift));
    const int page = a.table.at[b * a.table.sb + j];
    const bool there = page >= 0 && page < a.table.n_pages;
    float sum[8] = {};
    if (there && chunk < line) {
      const unsigned short* at = a.k.ptr + page * a.k.sp + (h * a.k.sh + d);
#pragma unroll 8
      for (int r = r0; r < n; r += step) {
        const u32x4 x = *(const u32x4*)(at + r * a.k.st);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum[2 * e] += T::up((unsigned short)x[e]);
          sum[2 * e + 1] += T::up((unsigned short)(x[e] >> 16));
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s_sum[tid][e] = sum[e];
    __syncthreads();
    if (r0 == 0 && there && chunk < line) {
      for (int g = 1; g < step; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += s_sum[tid + g * cols][e];
      const float count = (float)n;
      *(u32x4*)(a.means + page * a.means_sp + (h * a.means_sh + d)) =
          (u32x4){T::down2(sum[0] / count, sum[1] / count), T::down2(sum[2] / count, sum[3] / count), T::down2(sum[4] / count, sum[5] / count),
                  T::down2(sum[6] / count, sum[7] / count)};
    }
    __syncthreads();
  }
}

hipError_t launch_means(const MeansArgs& args, int dtype, hipStream_t stream) {
  MeansArgs a = args;
  const int line = a.H * a.D / 8;
  // neighbouring threads on as many chunks as leave less than half of the last workgroup's without one
  a.cols = 64;
  while (a.cols > 8 && line % a.cols != 0 && line % a.cols <= a.cols / 2) a.cols /= 2;
  const int wgs = a.B < 512 ? 512 : (a.B < 1024 ? a.B : 1024);
  void (*kernel)(MeansArgs) = dtype == RA_DTYPE_F16 ? means_kernel<F16> : means_kernel<BF16>;
  hipLaunchKernelGGL(kernel, dim3(wgs, (line + a.cols - 1) / a.cols), dim3(kMeanThreads), (a.B + 1) * sizeof(int), stream, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// choice of pages
// ---------------------------------------------------------------------------------------
// Scores: (sum of the group's queries) . (mean key), in 64 bits: products of 16-bit floats are exact there, and so are their sums but for
// extreme ranges, so that the order of pages does not depend on the order of a sum.  A score becomes a whole number of the same order.
// Sixteen lanes (eight, four for narrow heads) read a page's mean in one go, a wave 64 of them; their partial sums are exchanged so that each
// lane ends with the sums of its own.  A load takes several heads of a page beside each other, where there are several: 16 x 8 heads, 37 MB of means,
// 12.3 us, with a head alone in a load 16.5.  In 32 bits it would be 3 us less, and the choice would depend on the order of the sums.
constexpr int kScoreRows = 256;  // (page, head)s of a workgroup, 64 a wave
constexpr unsigned long long kForced = ~0ull, kNotThere = 0;  // (before and behind all numbers: that of -inf is larger than 0)
RA_DEV unsigned long long ordered(double x) {
  if (x != x) return kForced - 1;  // (not a number: before every number, as sorting has it)
  const unsigned long long u = __builtin_bit_cast(unsigned long long, x + 0.0);  // (-0 and 0 are equal)
  return u >> 63 ? ~u : u | 1ull << 63;
}
// Sums s[0 .. 2 O) over 2 O lanes, each of which keeps the one whose number is its own: half of them go to the partner, lane by lane bit.
template <int O, int N>
RA_DEV void exchange(double (&s)[N], int lane) {
  if constexpr (O > 0) {
    const bool up = lane & O;
#pragma unroll
    for (int i = 0; i < O; ++i) {
      const double keep = up ? s[i + O] : s[i], send = up ? s[i] : s[i + O];
      s[i] = keep + __shfl_xor(send, O, 64);
    }
    exchange<O / 2>(s, lane);
  }
}

template <class T, int D>
struct Scores {
  static constexpr int LPR = D == 32 ? 4 : (D == 64 ? 8 : 16);  // lanes of a row
  static constexpr int RPI = 64 / LPR, ITERS = LPR;             // rows a load, loads for 64 rows

  const SelectArgs& a;
  const int b, h, c, pages_i, sub_page;  // this lane's head, place in a row, pages a load and which of them
  const bool in_row;
  const unsigned short* q_at;
  u32x4 x[4];  // four of the group's queries

  // `hs` heads from `h0` on, of a page beside each other, then the next page
  RA_DEV Scores(const SelectArgs& args, int b_, int h0, int hs)
      : a(args), b(b_), h(h0 + lane() / LPR % hs), c(lane() % LPR), pages_i(RPI / hs), sub_page(lane() / LPR / hs), in_row(c * 8 < D),
        q_at(args.q + b_ * args.q_sb + (long long)h * args.G * args.q_sh + (in_row ? c * 8 : 0)) {}
  static RA_DEV int lane() { return threadIdx.x & 63; }
  RA_DEV void load_queries() {
#pragma unroll
    for (int g = 0; g < 4; ++g) x[g] = *(const u32x4*)(q_at + (long long)min(g, a.G - 1) * a.q_sh);
  }
  // The queries are there from here on: loaded where they are used, each would wait for all of the means.
  RA_DEV void have_queries() {
#pragma unroll
    for (int g = 0; g < 4; ++g) asm volatile("" : "+v"(x[g]));
  }
  RA_DEV int page_entry(int p0) const { return a.table.at[b * a.table.sb + min(p0 + lane(), a.table.width - 1)]; }

  // The number of page p0 + in_wave() for head h, of n pages; `mine`: page_entry(p0).
  RA_DEV int in_wave() const { return c * pages_i + sub_page; }
  RA_DEV unsigned long long number(int mine, int p0, int n) {
    u32x4 m[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      const int page = min(max(__shfl(mine, i * pages_i + sub_page, 64), 0), a.table.n_pages - 1);
      m[i] = *(const u32x4*)(a.means + page * a.means_sp + (h * a.means_sh + (in_row ? c * 8 : 0)));
      if constexpr (D == 96) m[i] = in_row ? m[i] : (u32x4){0, 0, 0, 0};
    }
    double q[8] = {};
    for (int g0 = 0; g0 < a.G; g0 += 4) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g0 + g >= a.G) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned y = in_row ? x[g][e] : 0u;
          q[2 * e] += (double)T::up((unsigned short)y);
          q[2 * e + 1] += (double)T::up((unsigned short)(y >> 16));
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (g0 + 4 < a.G) x[g] = *(const u32x4*)(q_at + (long long)min(g0 + 4 + g, a.G - 1) * a.q_sh);
    }
    double s[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      s[i] = 0.0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i] = __builtin_fma(q[2 * e], (double)T::up((unsigned short)m[i][e]), s[i]);
        s[i] = __builtin_fma(q[2 * e + 1], (double)T::up((unsigned short)(m[i][e] >> 16)), s[i]);
      }
    }
    exchange<LPR / 2>(s, c);  // (lane c of a row's lanes: the rows of load c)
    const int p = p0 + in_wave(), page = __shfl(mine, in_wave(), 64);
    if (page < 0 || page >= a.table.n_pages) return kNotThere;
    return p < a.first || p >= n - a.last ? kForced : ordered(s[0]);
  }
};
RA_DEV int row_pages(const SelectArgs& a, int length) { return pages_of(min(max(length, 0), a.table.width << a.table.shift), a.table.shift); }

template <class T, int D>
__global__ __launch_bounds__(256) void score_kernel(const SelectArgs a) {
  const int hs = a.heads, b = blockIdx.z, p0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / hs);
  Scores<T, D> scores(a, b, blockIdx.y * hs, hs);
  // the length, the pages and the queries are on their way together
  const int mine = scores.page_entry(p0), length = a.lengths[b];
  scores.load_queries();
  const int n = row_pages(a, length);
  scores.have_queries();
  if (p0 >= n || n <= a.count) return;  // (few pages: all of them, whatever their scores)
  const unsigned long long x = scores.number(mine, p0, n);
  const int p = p0 + scores.in_wave();
  if (p < n) a.keys[((long long)b * a.H + scores.h) * a.table.width + p] = x;
}

// The `count` largest of a row's numbers, ties from the lowest place, their places in order: the threshold by its digits of twelve bits (ten
// for few numbers) from the top, until all that share the digits found so far are taken; then every wave places what it takes of its part of the
// row.  Twelve bits: the first digit is a double's sign and exponent, and the second mostly settles it.  Bound by latency: some ten
// barriers, and few numbers between them: 128 of 4096 for 128 (row, head)s 6.3 us.  HELD: the row's numbers stay in registers, kHeld of a thread (read from the caches in every
// pass: 12; from shared memory: 11.5).
constexpr int kHeld = 8;
RA_DEV void take_all(const SelectArgs& a, int* out, int n) {
  for (int i = threadIdx.x; i < a.count; i += blockDim.x) out[i] = i < n ? i : -1;
}
// Of the numbers `load(place)`, places [0, n), n > a.count; a wave has places of its own, `rounds` times 64 of them.
template <int NT, bool HELD, class Load>
RA_DEV void choose(const SelectArgs& a, int* out, int n, int rounds, const unsigned long long (&held)[kHeld], Load load) {
  constexpr int WAVES = NT / 64, kDigitBits = NT > 256 ? 12 : 10, kDigits = 1 << kDigitBits, DPT = kDigits / NT;
  __shared__ int s_hist[kDigits], s_pick[3], s_above[WAVES], s_equal[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = rounds * 64, from = wave * part + lane, to = min(wave * part + part, n);
  // every number of this thread: place, number (places from `to` on: whatever lies there)
  auto each = [&](auto&& use) {
    if constexpr (HELD) {
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
        if (r < rounds) use(from + 64 * r, held[r]);
    } else {
      for (int r = 0; r < rounds && from - lane + 64 * r < n; ++r) use(from + 64 * r, load(from + 64 * r));
    }
  };
  // `known` bits from the top are those of the threshold; `need` of the numbers that have them are to be taken
  int known = 0, need = a.count, sharing = n;
  unsigned long long top = 0, mask = 0;
  while (known < 64 && need < sharing) {
    const int bits = min(kDigitBits, 64 - known), down = 64 - known - bits;
#pragma unroll
    for (int i = 0; i < DPT; ++i) s_hist[tid + i * NT] = 0;
    __syncthreads();
    each([&](int i, unsigned long long x) {
      if (i < to && (x & mask) == top) atomicAdd(&s_hist[(int)(x >> down) & ((1 << bits) - 1)], 1);
    });
    __syncthreads();
    // digits from the highest, neighbours in a thread; sums within a wave, then over the waves before it
    int c[DPT], sum = 0;
#pragma unroll
    for (int e = 0; e < DPT; ++e) {
      c[e] = s_hist[kDigits - 1 - DPT * tid - e];
      sum += c[e];
    }
    const int upto = scan_sum(sum);
    if (lane == 63) s_above[wave] = upto;
    __syncthreads();
    int above = upto - sum;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) above += w < wave ? s_above[w] : 0;
    if (above < need && above + sum >= need) {
#pragma unroll
      for (int e = 0; e < DPT; ++e) {
        if (above < need && above + c[e] >= need) {
          s_pick[0] = kDigits - 1 - DPT * tid - e;
          s_pick[1] = above;
          s_pick[2] = c[e];
        }
        above += c[e];
      }
    }
    __syncthreads();
    need -= s_pick[1];
    sharing = s_pick[2];
    top |= (unsigned long long)s_pick[0] << down;
    known += bits;
    mask = ~0ull << (64 - known);
  }
  int above = 0, equal = 0;
  each([&](int i, unsigned long long x) {
    above += __popcll(__ballot(i < to && (x & mask) > top));
    equal += __popcll(__ballot(i < to && (x & mask) == top));
  });
  __syncthreads();
  if (lane == 0) {
    s_above[wave] = above;
    s_equal[wave] = equal;
  }
  __syncthreads();
  above = equal = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    above += w < wave ? s_above[w] : 0;
    equal += w < wave ? s_equal[w] : 0;
  }
  const unsigned long long below = (1ull << lane) - 1;
  each([&](int i, unsigned long long x) {
    const bool gt = i < to && (x & mask) > top, eq = i < to && (x & mask) == top;
    const unsigned long long gts = __ballot(gt), eqs = __ballot(eq);
    const int my_gt = above + __popcll(gts & below), my_eq = equal + __popcll(eqs & below);
    if (gt || (eq && my_eq < need)) out[my_gt + min(my_eq, need)] = i;
    above += __popcll(gts);
    equal += __popcll(eqs);
  });
}

template <int NT, bool HELD>
__global__ __launch_bounds__(NT) void select_kernel(const SelectArgs a) {
  const int b = blockIdx.y, h = blockIdx.x, width = a.table.width;
  const unsigned long long* keys = a.keys + ((long long)b * a.H + h) * width;
  auto load = [&](int i) { return keys[min(i, width - 1)]; };
  // parts of the table's width: a thread's numbers are on their way together with the length
  const int rounds = (width + NT - 1) / NT, from = (threadIdx.x >> 6) * rounds * 64 + (threadIdx.x & 63);
  unsigned long long held[kHeld];
#pragma unroll
  for (int r = 0; r < kHeld; ++r) held[r] = HELD && width > a.count ? load(from + 64 * r) : 0;  // (else there is no workspace)
  const int n = row_pages(a, a.lengths[b]);
  int* out = a.pages + ((long long)b * a.H + h) * a.count;
  if (n <= a.count) take_all(a, out, n);
  else choose<NT, HELD>(a, out, n, rounds, held, load);
}

// Scores and choice of a (row, head) of few pages, which need no second kernel and no workspace.  In a graph, one kernel | two, us: 250 pages of 2 x 2 heads
// 4.9 | 7.1, 512 of 8 heads 8.6 | 9.2, of 64 x 8 16.2 | 22.3: a compute unit reads the 128 KB of 512 pages' means about as fast as a second kernel starts.
template <class T, int D>
__global__ __launch_bounds__(256) void few_kernel(const SelectArgs a) {
  __shared__ unsigned long long s_keys[kFewPages];
  const int b = blockIdx.y, h = blockIdx.x, wave = threadIdx.x >> 6;
  Scores<T, D> scores(a, b, h, 1);
  scores.load_queries();
  int mine = scores.page_entry(wave * 64);
  const int n = row_pages(a, a.lengths[b]);
  int* out = a.pages + ((long long)b * a.H + h) * a.count;
  if (n <= a.count) {
    take_all(a, out, n);
    return;
  }
  for (int p0 = wave * 64; p0 < n; p0 += 256) {
    if (p0 >= 256) {
      mine = scores.page_entry(p0);
      scores.load_queries();
    }
    scores.have_queries();
    const unsigned long long x = scores.number(mine, p0, n);
    if (p0 + scores.in_wave() < n) s_keys[p0 + scores.in_wave()] = x;
  }
  __syncthreads();
  const int rounds = (n + 255) / 256, from = wave * rounds * 64 + (threadIdx.x & 63);
  auto load = [&](int i) { return s_keys[min(i, n - 1)]; };
  unsigned long long held[kHeld];
#pragma unroll
  for (int r = 0; r < kHeld; ++r) held[r] = 64 * 4 * r < kFewPages ? load(from + 64 * r) : 0;
  choose<256, true>(a, out, n, rounds, held, load);
}

template <class T>
static void launch_score(const SelectArgs& args, hipStream_t stream) {
  SelectArgs a = args;
  // as many heads of a page in one load as its rows hold and as divide the heads (means of neighbouring heads mostly lie side by side)
  a.heads = a.D == 32 ? 16 : (a.D == 64 ? 8 : 4);
  while (a.H % a.heads != 0) a.heads /= 2;
  const int pages = kScoreRows / a.heads;
  const dim3 grid((a.table.width + pages - 1) / pages, a.H / a.heads, a.B);
  void (*kernel)(SelectArgs) = a.D == 32 ? score_kernel<T, 32> : a.D == 64 ? score_kernel<T, 64> : a.D == 96 ? score_kernel<T, 96> : score_kernel<T, 128>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a);
}
template <class T>
static void launch_few(const SelectArgs& a, hipStream_t stream) {
  void (*kernel)(SelectArgs) = a.D == 32 ? few_kernel<T, 32> : a.D == 64 ? few_kernel<T, 64> : a.D == 96 ? few_kernel<T, 96> : few_kernel<T, 128>;
  hipLaunchKernelGGL(kernel, dim3(a.H, a.B), dim3(256), 0, stream, a);
}
long long select_workspace(int width, long long rows) { return width <= kFewPages ? 0 : rows * width * (long long)sizeof(unsigned long long); }
hipError_t launch_select(const SelectArgs& a, int dtype, hipStream_t stream) {
  if (a.table.width <= kFewPages) {
    if (dtype == RA_DTYPE_F16) launch_few<F16>(a, stream);
    else launch_few<BF16>(a, stream);
    return hipGetLastError();
  }
  if (a.table.width > a.count) {  // (else every row has few pages)
    if (dtype == RA_DTYPE_F16) launch_score<F16>(a, stream);
    else launch_score<BF16>(a, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  // (four waves pass a barrier sooner than sixteen)
  if (a.table.width <= kHeld * 256) hipLaunchKernelGGL((select_kernel<256, true>), dim3(a.H, a.B), dim3(256), 0, stream, a);
  else if (a.table.width <= kHeld * 512) hipLaunchKernelGGL((select_kernel<512, true>), dim3(a.H, a.B), dim3(512), 0, stream, a);
  else if (a.table.width <= kHeld * 1024) hipLaunchKernelGGL((select_kernel<1024, true>), dim3(a.H, a.B), dim3(1024), 0, stream, a);
  else hipLaunchKernelGGL((select_kernel<1024, false>), dim3(a.H, a.B), dim3(1024), 0, stream, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// attention of one token per sequence
// ---------------------------------------------------------------------------------------
// The work of a call is one line of steps of 128 keys: row by row of the batch, head by head of the cache, along the sequence.  Every workgroup
// takes an equal stretch of it, so that rows of any lengths load the chip evenly; lengths are on the device, and each workgroup makes the
// line's prefix sums for itself.  A stretch that holds a (row, head) whole stores its output; parts of one go to memory as (maximum, sum,
// unnormalised output) in 32 bits and are joined by a second kernel.  Short rows (paged_shape): a workgroup of eight waves takes each (row, head)
// whole, and that is all.
// (of chosen pages all are looked at)
RA_DEV int first_key(const PagedArgs& a, int len) { return a.window > 0 && a.pages == nullptr ? max(len - a.window, 0) & ~31 : 0; }
RA_DEV int row_length(const PagedArgs& a, int b) { return min(max(a.lengths[b], 0), a.table.width << a.table.shift); }
// Pages of a row that are read, or looked at: no more than it has.
RA_DEV int row_entries(const PagedArgs& a, int len) { return min(pages_of(len, a.table.shift), a.pages != nullptr ? a.count : a.table.width); }
template <int STEP>
RA_DEV int row_steps(const PagedArgs& a, int len) {
  if (a.pages != nullptr) len = row_entries(a, len) << a.table.shift;
  return max((len - first_key(a, len) + STEP - 1) / STEP, 1);  // (one for an empty row: its output is stored too)
}
RA_DEV unsigned start_of(unsigned wg, unsigned whole, unsigned rest) { return wg * whole + min(wg, rest); }
RA_DEV unsigned holder_of(unsigned step, unsigned whole, unsigned rest) {
  const unsigned ahead = rest * (whole + 1);
  return step < ahead ? step / (whole + 1) : rest + (step - ahead) / whole;
}

// (a maximum of -inf beside a sum: all scores that count are not numbers)
template <class T>
RA_DEV float logsumexp_of(float top, float sum) {
  return ((top == RA_NEG_INF ? 0.f : top) - T::kLift + __builtin_amdgcn_logf(sum)) * kLn2;
}

// A wave's 32 keys and values on their way.  Both are loaded with neighbouring lanes on neighbouring 16 bytes of a row: a load whose lanes 0 .. 15 are on
// rows of their own, as the matrix instruction wants keys, takes a cache lookup for each of them (a compute unit gets 38 GB/s so, and 148 from whole
// rows).  Keys then pass through the wave's own piece of shared memory: instruction i of a half writes the 16-byte chunks 64 i .. 64 i + 63 of its
// sixteen rows, and lane l reads chunks l / 16 + 4 s of key l % 16, the first operand.  Of values lane l holds, of D / 16 elements from (l % 16) D / 16,
// the eight keys whose weights it gets from the scores' product: 4 (l / 16) + 0 .. 3 of each half.  Nothing is shared between waves but their ends.
template <int D>
struct KeyTile {
  u32x4 k[2][D / 32];
  unsigned v[8][D / 32];
};
// The place of a key row's chunk among the row's: sixteen rows' chunks of one number lie in different banks.
template <int D>
RA_DEV int chunk_place(int row, int chunk) {
  if constexpr (D == 128) return chunk ^ row;
  if constexpr (D == 96) return (chunk + row / 4) % 12;
  if constexpr (D == 64) return chunk ^ row / 2;
  return chunk ^ row / 4;
}

// STREAM: the caches are not to keep it, as they cannot keep what a large call reads once (64 x 8 heads, 2.06 GB: 336 us against 367; 231 MB 48.6 against 54.0); a small one's
// keys may be there from the step before (1000 x 8 heads, whole: 4 us more with the hint where they would have been).
// (an overload for each width: a template's parameter would not keep that rows are aligned to four bytes only)
template <bool STREAM>
RA_DEV u32x4 load_row(const u32x4* at) {
  return STREAM ? __builtin_nontemporal_load(at) : *at;
}
template <bool STREAM>
RA_DEV u32x3a load_row(const u32x3a* at) {
  return STREAM ? __builtin_nontemporal_load(at) : *at;
}
template <bool STREAM>
RA_DEV u32x2a load_row(const u32x2a* at) {
  return STREAM ? __builtin_nontemporal_load(at) : *at;
}
template <bool STREAM>
RA_DEV unsigned load_row(const unsigned* at) {
  return STREAM ? __builtin_nontemporal_load(at) : *at;
}
template <int D, bool STREAM>
RA_DEV void load_values(unsigned (&v)[D / 32], const unsigned short* at) {
  if constexpr (D == 128) {
    const u32x4 x = load_row<STREAM>((const u32x4*)at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i];
  } else if constexpr (D == 96) {
    const u32x3a x = load_row<STREAM>((const u32x3a*)at);
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] = x[i];
  } else if constexpr (D == 64) {
    const u32x2a x = load_row<STREAM>((const u32x2a*)at);
    v[0] = x[0];
    v[1] = x[1];
  } else {
    v[0] = load_row<STREAM>((const unsigned*)at);
  }
}

constexpr int kPieces = 3;  // of a weight
constexpr int kEntries = 1024, kNearRows = 1024;  // of a stretch's pages, of the rows' lengths in shared memory
constexpr int kNowhere = 0x7ff00000;  // (a position behind every sequence, of 2^30 tokens at most; a page and a tile on top of it fit 32 bits)

// HBM bound: the matrix unit multiplies sixteen rows however few there are, and is busy for a twelfth of the time.  64 x 8 heads, 2.06 GB, 331 us (6.2 TB/s), 32 x
// 131071 keys, 2.15 GB, 328 (6.5); 16 x 16 heads, 231 MB, 44, of which 4 pass before the first keys arrive.  A call on 1000 keys of 8 heads,
// D=64, is 8.5 us of one workgroup per head: what a compute unit alone gets from memory.
template <class T, int D, bool ALIBI, bool WHOLE>
__global__ __launch_bounds__(WHOLE ? 512 : 256, 2) void paged_kernel(const PagedArgs a) {
  constexpr int WAVES = WHOLE ? 8 : 4, THREADS = 64 * WAVES, STEP = 32 * WAVES;
  constexpr int KS = D / 32;  // matrix instructions of a score, words of a lane's value row
  constexpr int DPL = D / 16;  // elements of a lane's value row
  constexpr int CHUNKS = D / 8;  // of 16 bytes in a row
  extern __shared__ int s_first[];
  __shared__ int red[WAVES][1];
  __shared__ int s_page[kEntries], s_pos[kEntries], s_len[WHOLE ? 1 : kNearRows];
  __shared__ float s_m[WAVES][16], s_l[WAVES][16];
  // the waves' keys, and when all are through their outputs, elements in the order of the lanes' registers: 16 i + m is element m D / 16 + i
  __shared__ union {
    u32x4 k[WAVES][2][16 * CHUNKS];
    float o[WAVES][16][D + 4];
  } s_tile;
  auto& s_o = s_tile.o;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int units = a.H * a.tiles;  // of a row
  // this lane's chunks of a half's rows: where they are in the pool, where they go, and where its operands are
  int k_from[KS], k_to[KS], k_at[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int row = (64 * i + lane) / CHUNKS, chunk = (64 * i + lane) % CHUNKS;
    k_from[i] = row * a.k.st + chunk * 8;
    k_to[i] = row * CHUNKS + chunk_place<D>(row, chunk);
    k_at[i] = col * CHUNKS + chunk_place<D>(col, 4 * i + grp);
  }
  unsigned whole = 0, rest = 0, begin = 0, end = 1;
  if constexpr (!WHOLE) {
    scan_rows<THREADS, 1>(
        a.B,
        [&](int b, int (&x)[1]) {
          const int len = row_length(a, b);
          if (b < kNearRows) s_len[b] = len;
          x[0] = row_steps<STEP>(a, len);
        },
        {s_first}, red);
    const unsigned total = (unsigned)s_first[a.B] * (unsigned)units;
    const unsigned n_wg = min((unsigned)a.n_wg, max(total / kStepsEach, (unsigned)kFewWorkgroups));
    whole = total / n_wg;
    rest = total % n_wg;
    if (blockIdx.x >= n_wg) return;
    begin = start_of(blockIdx.x, whole, rest);
    end = start_of(blockIdx.x + 1, whole, rest);
  }
  unsigned at = begin;
  const int size = 1 << a.table.shift;
  while (at < end) {
    // the (row, head) that the stretch is in, and which of its steps
    int b, len;
    unsigned unit, unit0, steps, upto;
    if constexpr (WHOLE) {
      b = blockIdx.y;
      unit = blockIdx.x;
      len = row_length(a, b);
      steps = row_steps<STEP>(a, len);
      unit0 = 0;
      upto = steps;
    } else {
      b = __builtin_amdgcn_readfirstlane(row_of(s_first, a.B, (int)(at / (unsigned)units)));
      len = __builtin_amdgcn_readfirstlane(b < kNearRows ? s_len[b] : row_length(a, b));
      const unsigned row0 = (unsigned)s_first[b] * units;
      steps = (unsigned)__builtin_amdgcn_readfirstlane(s_first[b + 1] - s_first[b]);
      unit = __builtin_amdgcn_readfirstlane((at - row0) / steps);
      unit0 = row0 + unit * steps;
      upto = min(end, unit0 + steps);
    }
    const int h = a.tiles == 1 ? (int)unit : (int)unit / a.tiles, tile = (int)unit - h * a.tiles;
    const int heads = min(a.G - tile * 16, 16);  // query heads of this unit
    const long long head0 = (long long)b * a.H * a.G + h * a.G + tile * 16;
    const int low = a.window > 0 ? max(len - a.window, 0) : 0, key0 = first_key(a, len);
    u32x4 q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
      q[s] = col < heads ? *(const u32x4*)(a.q + b * a.q_sb + (long long)(h * a.G + tile * 16 + col) * a.q_sh + s * 32 + grp * 8) : (u32x4){0, 0, 0, 0};
    float slope = 0.f;
    if constexpr (ALIBI) slope = col < heads ? a.slopes[h * a.G + tile * 16 + col] * kLog2e : 0.f;
    float m = RA_NEG_INF, l = 0.f;
    f32x4 o[DPL];
#pragma unroll
    for (int i = 0; i < DPL; ++i) o[i] = (f32x4){0.f, 0.f, 0.f, 0.f};

    const int n_entries = row_entries(a, len);
    // kEntries pages at a time
    unsigned step = at - unit0;
    const unsigned step_end = upto - unit0;
    while (step < step_end) {
      const int from_key = key0 + (int)step * STEP, entry0 = from_key >> a.table.shift;
      const unsigned fit = (unsigned)(((entry0 + kEntries) << a.table.shift) - from_key) / STEP;
      const unsigned chunk_end = min(step_end, step + fit);
      const int n_here = min(((key0 + (int)chunk_end * STEP - 1) >> a.table.shift) - entry0 + 1, kEntries);
      __syncthreads();  // (the entries of the chunk before have been read)
      for (int i = tid; i < n_here; i += THREADS) {
        const int e = entry0 + i;
        int logical = e < n_entries ? e : -1;
        if (a.pages != nullptr && logical >= 0) logical = a.pages[((long long)b * a.H + h) * a.count + e];
        int page = logical >= 0 && logical < a.table.width ? a.table.at[b * a.table.sb + logical] : -1;
        const bool there = page >= 0 && page < a.table.n_pages;
        s_page[i] = there ? page : 0;
        s_pos[i] = there ? logical << a.table.shift : kNowhere;
      }
      __syncthreads();
      // A step's keys are replaced by the next one's as soon as they are in shared memory, its values after the product with the weights: one is
      // always on its way while the other is used, in the registers of a single step.
      KeyTile<D> x;
      int p[2];
      auto load = [&](unsigned s, bool values) {
        const int key = key0 + (int)s * STEP + wave * 32;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int kt = key + 16 * t, off = kt & (size - 1);
          const long long page = __builtin_amdgcn_readfirstlane(s_page[(kt >> a.table.shift) - entry0]);
          if (values) {
            const unsigned short* vp = a.v.ptr + page * a.v.sp + (off * a.v.st + h * a.v.sh);
#pragma unroll
            for (int j = 0; j < 4; ++j) load_values<D, !WHOLE>(x.v[4 * t + j], vp + ((4 * grp + j) * a.v.st + col * DPL));
          } else {
            const unsigned short* kp = a.k.ptr + page * a.k.sp + (off * a.k.st + h * a.k.sh);
#pragma unroll
            for (int i = 0; i < KS; ++i) x.k[t][i] = load_row<!WHOLE>((const u32x4*)(kp + k_from[i]));
          }
        }
      };
      load(step, false);
      load(step, true);
      for (; step < chunk_end; ++step) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int kt = key0 + (int)step * STEP + wave * 32 + 16 * t;
          p[t] = __builtin_amdgcn_readfirstlane(s_pos[(kt >> a.table.shift) - entry0]) + (kt & (size - 1));
        }
        // (a wave's accesses to shared memory are done in their order: the fences keep the compiler to it, and cost nothing)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < KS; ++i) s_tile.k[wave][t][k_to[i]] = x.k[t][i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (step + 1 < chunk_end) load(step + 1, false);
        float w[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < KS; ++i) c = T::mfma(s_tile.k[wave][t][k_at[i]], q[i], c);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            w[4 * t + r] = c[r] * a.scale2;
            if constexpr (ALIBI) w[4 * t + r] -= slope * (float)(len - 1 - p[t] - 4 * grp - r);
          }
        }
        const bool inside = p[0] >= low && p[0] + 16 <= len && p[1] >= low && p[1] + 16 <= len;
        if (!inside) {
          // What is masked may hold anything: its score is replaced, and its value too (0 times infinity is not 0).
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at_key = p[j >> 2] + 4 * grp + (j & 3);
            const bool on = at_key >= low && at_key < len;
            w[j] = on ? w[j] : RA_NEG_INF;
#pragma unroll
            for (int i = 0; i < KS; ++i) x.v[j][i] = on ? x.v[j][i] : 0u;
          }
        }
        float top = fmaxf(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])), fmaxf(fmaxf(w[4], w[5]), fmaxf(w[6], w[7])));
        top = max_of_rows(top);
        if (__any(top > m)) {
          const float next = fmaxf(m, top), keep = next == RA_NEG_INF ? 1.f : __builtin_amdgcn_exp2f(m - next);
          m = next;
          l *= keep;
#pragma unroll
          for (int i = 0; i < DPL; ++i) o[i] *= keep;
        }
        const float base = m == RA_NEG_INF ? 0.f : m - T::kLift;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          w[j] = __builtin_amdgcn_exp2f(w[j] - base);
          l += w[j];
        }
        // A weight goes in as three pieces, each of what the ones before lack of it, through the matrix unit, which has the time: all its 24 bits, so that the output
        // is off by its own rounding and by sums in 32 bits.  (Two pieces of bf16 left 2^-17 of a weight: one output in 500 was the neighbour of the nearest number.)
        // The first two are cut off, not rounded, and what is left is made no less than 2^-31 of the weight (fp16: than 2^-24, its least, 2^-39 of the largest weight): pieces
        // of 0 or below it would make NaN of an infinite value.
        u32x4 piece[kPieces];
        float left[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) left[j] = w[j];
#pragma unroll
        for (int n = 0; n < kPieces; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) piece[n][j] = n + 1 < kPieces ? T::cut2(left[2 * j], left[2 * j + 1]) : T::down2(left[2 * j], left[2 * j + 1]);
#pragma unroll
          for (int j = 0; j < 8; ++j) left[j] = T::rest(w[j], left[j] - T::up((unsigned short)(piece[n][j / 2] >> (j & 1 ? 16 : 0))));
        }
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
          const unsigned pick = i & 1 ? 0x07060302u : 0x05040100u;
          u32x4 vt;
#pragma unroll
          for (int j = 0; j < 4; ++j) vt[j] = __builtin_amdgcn_perm(x.v[2 * j + 1][i >> 1], x.v[2 * j][i >> 1], pick);
#pragma unroll
          for (int n = 0; n < kPieces; ++n) o[i] = T::mfma(vt, piece[n], o[i]);
        }
        if (step + 1 < chunk_end) load(step + 1, true);
      }
    }

    // The waves' parts.  What runs once is short: its instructions come from memory, and take longer than what they do.
    l = sum_of_rows(l);
    __syncthreads();  // (the sums of the unit before have been read)
    if (grp == 0) {
      s_m[wave][col] = m;
      s_l[wave][col] = l;
    }
    if (col < heads) {
#pragma unroll
      for (int i = 0; i < DPL; ++i) *(f32x4*)&s_o[wave][col][16 * i + 4 * grp] = o[i];
    }
    __syncthreads();
    const bool complete = at == unit0 && upto == unit0 + steps;
    const long long slot = 2ll * blockIdx.x + (at != begin);
    if (!WHOLE && at == unit0 && tid == 0) {
      // where the join finds the parts: a workgroup's first unit has its first place, so all but the first part lie in even ones
      const unsigned last = complete ? blockIdx.x : holder_of(unit0 + steps - 1, whole, rest);
      a.where[b * units + (int)unit] = make_int2((int)slot, (int)(last - blockIdx.x) + 1);
    }
    // a thread for D / 16 neighbouring elements of a query head
    if (tid < heads * 16) {
      const int r = tid / 16, c = tid % 16;
      float top = RA_NEG_INF, sum = 0.f, x[DPL];
#pragma unroll 4
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, s_m[w][r]);
      const float base = top == RA_NEG_INF ? 0.f : top;  // (a wave without a score has a maximum of -inf, and a weight of 0)
#pragma unroll
      for (int i = 0; i < DPL; ++i) x[i] = 0.f;
#pragma unroll 4
      for (int w = 0; w < WAVES; ++w) {
        const float part = __builtin_amdgcn_exp2f(s_m[w][r] - base);
        sum += s_l[w][r] * part;
#pragma unroll
        for (int i = 0; i < DPL; ++i) x[i] += s_o[w][r][16 * i + c] * part;
      }
      if (WHOLE || complete) {
        // (a row without a key has a sum of 0; scores that are not numbers are in no maximum, but in the sum)
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        unsigned* out = (unsigned*)(a.out + (head0 + r) * D + c * DPL);
#pragma unroll
        for (int i = 0; i < DPL; i += 2) out[i / 2] = T::down2(x[i] * inv, x[i + 1] * inv);
        if (c == 0) a.lse[head0 + r] = sum == 0.f ? RA_NEG_INF : logsumexp_of<T>(top, sum);
      } else {
        float* p = a.part + (slot * kPartRows + r) * D + c * DPL;
#pragma unroll
        for (int i = 0; i < DPL; ++i) p[i] = x[i];
        if (c == 0) a.stats[slot * kPartRows + r] = make_float2(top, sum);
      }
    }
    at = WHOLE ? end : upto;
  }
}

// The parts of a (row, query head): a workgroup each, threads on neighbouring elements and on different parts.  Latency bound: a part's statistics and
// its elements are on their way together, for 64 parts at a time: 2.6 us for 60 (row, head)s, 4.1 for 2048.
template <class T, int D>
__global__ __launch_bounds__(256) void join_kernel(const PagedArgs a) {
  constexpr int COLS = D / 4, GROUPS = 256 / COLS, MOST = (64 + GROUPS - 1) / GROUPS;
  __shared__ float s_sum[GROUPS][D];
  const int tid = threadIdx.x, lane = tid & 63;
  const int b = blockIdx.y, head = blockIdx.x, h = head / a.G, g = head % a.G, r = g % 16;
  const int2 where = a.where[b * a.H * a.tiles + h * a.tiles + g / 16];
  const int parts = where.y;
  if (parts <= 1) return;
  auto place = [&](int i) { return (long long)(i == 0 ? where.x : (where.x & ~1) + 2 * i) * kPartRows + r; };
  const int c = tid % COLS, p0 = tid / COLS;
  float top = RA_NEG_INF, sum = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < parts; i0 += 64) {
    const int n = min(parts - i0, 64);
    const float2 st = a.stats[place(i0 + min(lane, n - 1))];
    f32x4 y[MOST];
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
      const int i = p0 + j * GROUPS;
      y[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
      if (p0 < GROUPS && i < n) y[j] = *(const f32x4*)(a.part + place(i0 + i) * D + 4 * c);
    }
    const float next = fmaxf(max_of_wave(lane < n ? st.x : RA_NEG_INF), top);
    const float keep = top == RA_NEG_INF ? 0.f : __builtin_amdgcn_exp2f(top - next);
    const float w = lane < n && st.x != RA_NEG_INF ? __builtin_amdgcn_exp2f(st.x - next) : 0.f;
    const float s = sum_of_wave(lane < n ? w * st.y : 0.f);
    // (what is not a number stays so under a weight of 0)
    sum = sum * keep + s;
    x *= keep;
    top = next;
#pragma unroll
    for (int j = 0; j < MOST; ++j) x += __shfl(w, (p0 + j * GROUPS) & 63, 64) * y[j];
  }
  if (p0 < GROUPS) *(f32x4*)&s_sum[p0][4 * c] = x;
  __syncthreads();
  const long long at = (long long)b * a.H * a.G + head;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (tid < D / 2) {
    float y = 0.f, z = 0.f;
#pragma unroll
    for (int p = 0; p < GROUPS; ++p) {
      y += s_sum[p][2 * tid];
      z += s_sum[p][2 * tid + 1];
    }
    *(unsigned*)(a.out + at * D + 2 * tid) = T::down2(y * inv, z * inv);
  }
  if (tid == 0) a.lse[at] = sum == 0.f ? RA_NEG_INF : logsumexp_of<T>(top, sum);
}

// The workspace: parts, their statistics, and where those of each (row, head) are.
static long long part_bytes(int n_wg, int D) { return 2ll * n_wg * kPartRows * D * (long long)sizeof(float); }
static long long stat_bytes(int n_wg) { return 2ll * n_wg * kPartRows * (long long)sizeof(float2); }
PagedShape paged_shape(long long keys, long long units, int D) {
  const long long steps = (keys + kStepKeys - 1) / kStepKeys, most = steps * units;
  if (keys * D <= kWholeSize || (keys <= kWholeKeys && units >= kWholeUnits)) return {(int)units, true, 0};
  // (as the kernel has it, of the steps that there are at most)
  const long long wanted = most / kStepsEach > kFewWorkgroups ? most / kStepsEach : kFewWorkgroups, cap = most < kPagedWorkgroups ? most : kPagedWorkgroups;
  const int n_wg = (int)(wanted < cap ? wanted : cap);
  return {n_wg, false, part_bytes(n_wg, D) + stat_bytes(n_wg) + units * (long long)sizeof(int2)};
}

template <class T, int D, bool ALIBI>
static hipError_t launch_paged_of(PagedArgs& a, const PagedShape& shape, void* workspace, hipStream_t stream) {
  a.n_wg = shape.workgroups;
  if (shape.whole) {
    hipLaunchKernelGGL((paged_kernel<T, D, ALIBI, true>), dim3(a.H * a.tiles, a.B), dim3(512), 0, stream, a);
    return hipGetLastError();
  }
  a.part = static_cast<float*>(workspace);
  a.stats = reinterpret_cast<float2*>(static_cast<char*>(workspace) + part_bytes(a.n_wg, D));
  a.where = reinterpret_cast<int2*>(static_cast<char*>(workspace) + part_bytes(a.n_wg, D) + stat_bytes(a.n_wg));
  hipLaunchKernelGGL((paged_kernel<T, D, ALIBI, false>), dim3(a.n_wg), dim3(256), (a.B + 1) * sizeof(int), stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((join_kernel<T, D>), dim3(a.H * a.G, a.B), dim3(256), 0, stream, a);
  return hipGetLastError();
}
template <class T>
static hipError_t launch_paged_type(PagedArgs& a, int D, const PagedShape& shape, void* workspace, hipStream_t stream) {
  const bool alibi = a.slopes != nullptr;
  switch (D) {
    case 32: return alibi ? launch_paged_of<T, 32, true>(a, shape, workspace, stream) : launch_paged_of<T, 32, false>(a, shape, workspace, stream);
    case 64: return alibi ? launch_paged_of<T, 64, true>(a, shape, workspace, stream) : launch_paged_of<T, 64, false>(a, shape, workspace, stream);
    case 96: return alibi ? launch_paged_of<T, 96, true>(a, shape, workspace, stream) : launch_paged_of<T, 96, false>(a, shape, workspace, stream);
    default: return alibi ? launch_paged_of<T, 128, true>(a, shape, workspace, stream) : launch_paged_of<T, 128, false>(a, shape, workspace, stream);
  }
}
hipError_t launch_paged(PagedArgs& a, int D, int dtype, const PagedShape& shape, void* workspace, hipStream_t stream) {
  return dtype == RA_DTYPE_F16 ? launch_paged_type<F16>(a, D, shape, workspace, stream) : launch_paged_type<BF16>(a, D, shape, workspace, stream);
}

// ---------------------------------------------------------------------------------------
// a few numbers from the host
// ---------------------------------------------------------------------------------------
// A copy from pageable memory waits for the stream and cannot be captured; a kernel's arguments are copied by the launch itself.  Up to 4 KB of them; one
// launch for 512 numbers, an empty kernel's time: a call with 12 slopes on the host takes 13.2 us, with slopes on the device 11.0, with such a copy 24.5.
constexpr int kPut = 512;
struct PutArgs {
  float* to;
  int n;
  float x[kPut];
};
__global__ __launch_bounds__(kPut) void put_kernel(const PutArgs a) {
  if ((int)threadIdx.x < a.n) a.to[threadIdx.x] = a.x[threadIdx.x];
}
hipError_t launch_put(const float* values, int n, float* to, hipStream_t stream) {
  PutArgs a;
  for (int i = 0; i < n; i += kPut) {
    a.to = to + i;
    a.n = n - i < kPut ? n - i : kPut;
    for (int j = 0; j < kPut; ++j) a.x[j] = j < a.n ? values[i + j] : 0.f;
    hipLaunchKernelGGL(put_kernel, dim3(1), dim3(kPut), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ra
