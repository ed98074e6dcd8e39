// Device code of the terms that take arguments of their own (TermArgs): the relative position bias by buckets, and dropout.
#pragma once
#include <type_traits>

#include "ra_launch.h"

namespace ra {

// ------------------------------------------------------------------------------------------------
// Dropout.  A weight (query i, key j) of head hh (batch * heads + head) has 16 bits of a counter-based generator: Philox 4x32 of seven rounds
// (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011: the fewest that pass all of their tests) with the
// seed as key and the counter (j / 2, i / 4, hh, 0); query i's word is the (i % 4)-th, an even key's half the low one.  A call serves eight weights
// whichever side the kernel's lanes own: four neighbouring lanes with a query each exchange words, and two with a key each halves.
// Vector issue bounds the kernels with dropout.  16 heads of 8192, causal, us, without | with: D=128 forward 322 | 390 (705 TFLOP/s), backward 838 | 1037.
// ------------------------------------------------------------------------------------------------
constexpr unsigned kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u, kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;
RA_DEV unsigned xor3(unsigned a, unsigned b, unsigned c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
// The r-th round (of 1 .. 7) on the words c; k0, k1: the seed.
RA_DEV void philox_round(int r, unsigned (&c)[4], unsigned k0, unsigned k1) {
  const unsigned long long a = (unsigned long long)c[0] * kPhiloxM0, b = (unsigned long long)c[2] * kPhiloxM1;
  c[0] = xor3((unsigned)(b >> 32), c[1], k0 + (r - 1) * kPhiloxW0);
  c[1] = (unsigned)b;
  c[2] = xor3((unsigned)(a >> 32), c[3], k1 + (r - 1) * kPhiloxW1);
  c[3] = (unsigned)a;
}
// The words c of four neighbouring lanes turned round, through a kilobyte of LDS that is the wave's own: word x of a lane becomes the lane's own word of
// the x-th lane.  (In registers that is sixteen vector instructions, of some 75 that dropout costs a lane's eight weights; LDS has room beside the tiles'
// operands, and gives all of its banks to either side.)  No barrier: a wave's LDS instructions are carried out in order.
struct WordTurn {
  unsigned *to, *from;
  RA_DEV void init(unsigned* lds, int lane) {
    to = lds + 4 * ((lane >> 2) + 16 * (lane & 3));
    from = lds + 4 * (lane >> 2) + (lane & 3);
  }
  RA_DEV void run(unsigned (&w)[4], const unsigned (&c)[4]) const {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    *(u32x4*)to = (u32x4){c[0], c[1], c[2], c[3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int x = 0; x < 4; ++x) w[x] = from[64 * x];
  }
};
// A call in steps, which the kernels lay between their matrix instructions: a round waits for the one before, and a wave that makes them in one go
// waits with it.  What the first rounds leave to do where a lane keeps its query (two of fourteen products are the same in every call) ...
struct PhiloxRow {
  static constexpr int kSteps = 6;
  unsigned a_high, a_low;  // of the second round's first product, the high word with its key
  static RA_DEV int pair(int lane) { return 2 * (lane >> 5) + 4 * ((lane >> 1) & 1) + (lane & 1); }  // of the sixteen keys of a group: where its call's two are
  RA_DEV void init(unsigned q_group, unsigned hh, unsigned k0, unsigned k1) {
    const unsigned long long b = (unsigned long long)hh * kPhiloxM1;
    const unsigned long long a = (unsigned long long)((unsigned)(b >> 32) ^ q_group ^ k0) * kPhiloxM0;
    a_high = (unsigned)(a >> 32) ^ (k1 + kPhiloxW1);
    a_low = (unsigned)a;
  }
  RA_DEV void step(int i, unsigned (&c)[4], unsigned k_pair, unsigned hh, unsigned k0, unsigned k1) const {
    asm volatile("" : "+s"(k0), "+s"(k1));  // (the keys of the rounds are made again, not kept: scalar registers are short)
    if (i > 0) return philox_round(i + 2, c, k0, k1);
    const unsigned long long a = (unsigned long long)k_pair * kPhiloxM0;
    const unsigned long long b = (unsigned long long)((unsigned)(a >> 32) ^ k1) * kPhiloxM1;
    c[0] = xor3((unsigned)(b >> 32), hh * kPhiloxM1, k0 + kPhiloxW0);
    c[1] = (unsigned)b;
    c[2] = a_high ^ (unsigned)a;
    c[3] = a_low;
  }
};
// ... and where it keeps its key (four, in the two calls for a block; kept through the loop they cost the backward's kernels spills).
struct PhiloxKey {
  static constexpr int kSteps = 5;
  unsigned a_low, b_low, a3_high, a3_low;  // of the first round's and the second's products, with keys; of the third's first
  RA_DEV void init(unsigned k_pair, unsigned hh, unsigned k0, unsigned k1) {
    const unsigned long long a = (unsigned long long)k_pair * kPhiloxM0;
    const unsigned long long b = (unsigned long long)((unsigned)(a >> 32) ^ k1) * kPhiloxM1;
    a_low = (unsigned)a ^ (k1 + kPhiloxW1);
    b_low = (unsigned)b ^ (k0 + 2 * kPhiloxW0);
    const unsigned long long a3 = (unsigned long long)((unsigned)(b >> 32) ^ (hh * kPhiloxM1) ^ (k0 + kPhiloxW0)) * kPhiloxM0;
    a3_high = (unsigned)(a3 >> 32) ^ (k1 + 2 * kPhiloxW1);
    a3_low = (unsigned)a3;
  }
  RA_DEV void step(int i, unsigned (&c)[4], unsigned q_group, unsigned hh, unsigned k0, unsigned k1) const {
    asm volatile("" : "+s"(k0), "+s"(k1));
    if (i > 0) return philox_round(i + 3, c, k0, k1);
    const unsigned first = (unsigned)(((unsigned long long)hh * kPhiloxM1) >> 32) ^ k0;
    const unsigned long long a = (unsigned long long)(q_group ^ first) * kPhiloxM0;
    const unsigned long long b = (unsigned long long)((unsigned)(a >> 32) ^ a_low) * kPhiloxM1;
    c[0] = (unsigned)(b >> 32) ^ b_low;
    c[1] = (unsigned)b;
    c[2] = a3_high ^ (unsigned)a;
    c[3] = a3_low;
  }
};

template <int CTRL>
RA_DEV unsigned lane_dpp(unsigned x) {  // (patterns that read every lane)
  return (unsigned)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
}
// All ones in the lanes whose number has the bit, and a choice by such a mask.
RA_DEV unsigned lane_bit(int lane, int bit) { return (unsigned)((int)((unsigned)lane << (31 - bit)) >> 31); }
RA_DEV unsigned choose(unsigned mask, unsigned a, unsigned b) {
  unsigned x = (mask & a) | (~mask & b);
  asm("" : "+v"(x));  // (one register is kept, not the two sides and their merge in every use)
  return x;
}
// Whether the weight of a word's half stays.
RA_DEV bool stays_low(unsigned w, unsigned drop) { return (unsigned short)w >= (unsigned short)drop; }
RA_DEV bool stays_high(unsigned w, unsigned drop) { return w >= drop << 16; }
// ... as a mask of lanes, to be used more than once: such a mask is kept out of VCC, which a v_cndmask reads in 4 cycles right behind the compare and in
// some 20 every further time (any other scalar pair: 4).  (Compares and choices are the compiler's, which places the waits between a vector instruction that
// writes a scalar pair, an exponential or a matrix instruction and the one that reads it; the empty statement keeps the pair.)
typedef unsigned long long lane_mask;
RA_DEV lane_mask lanes(bool stays) {
  lane_mask m = __builtin_amdgcn_ballot_w64(stays);
  asm("" : "+s"(m));
  return m;
}
RA_DEV lane_mask lanes_low(unsigned w, unsigned drop) { return lanes(stays_low(w, drop)); }
RA_DEV lane_mask lanes_high(unsigned w, unsigned drop) { return lanes(stays_high(w, drop)); }
RA_DEV float where(lane_mask m, float a, float b) { return __builtin_amdgcn_inverse_ballot_w64(m) ? a : b; }
RA_DEV float where_or_0(lane_mask m, float a) { return where(m, a, 0.f); }
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
// 1 in the halves of two 16-bit values that are at least `least`, which is 1 or more
RA_DEV u16x2 at_least(unsigned w, unsigned least) {
  const unsigned short most = least - 1;
  unsigned d = __builtin_bit_cast(unsigned, __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, w), u16x2{most, most}));
  // (by name: the compiler makes two compares, two choices and a merge of it.  Reads and writes one vector register, of a packed subtraction: no waits.)
  asm("v_pk_min_u16 %0, %0, 1 op_sel_hi:[1,0]" : "+v"(d));
  return __builtin_bit_cast(u16x2, d);
}
RA_DEV unsigned times_pair(unsigned x, unsigned y) {
  return __builtin_bit_cast(unsigned, (u16x2)(__builtin_bit_cast(u16x2, x) * __builtin_bit_cast(u16x2, y)));
}
// Two 16-bit elements, of which those stay whose halves of `w` do.
RA_DEV unsigned keep_pair(unsigned pair, unsigned w, unsigned drop) {
  return times_pair(pair, __builtin_bit_cast(unsigned, at_least(w, drop)));
}

// The seed's words, as uniform values.
RA_DEV void load_seed(const TermArgs& t, unsigned& k0, unsigned& k1) {
  const unsigned long long s = t.seed_at != nullptr ? *t.seed_at : t.seed;
  k0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)s);
  k1 = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(s >> 32));
}

// ------------------------------------------------------------------------------------------------
// The relative bias.  It is a function of the distance d = key - query, constant from the last bucket's start on (and, one-sided, from 0 on): a
// block of 32 x 32 scores that lies there takes one number into its exponents, and no other work.  For the tiles on the way the
// workgroup writes the values of a tile's distances to LDS, one a thread, while the tile is on its way, and a score reads its own.  A token on 32768
// keys (4 batch rows of 16 heads, padded, D=128) runs at what memory gives, the others are bound as the kernels without it: 16 heads of 2 x 4096, causal, D=64, us, without | with: backward
// 259 | 293, forward 105 | 141 (106 but for the second product of the output, see fwd_pair_kernel).
// ------------------------------------------------------------------------------------------------
// Buckets in the order of d: the far past first, the far future last (one-sided: bucket 0 last).
RA_DEV int ordered_bucket(const int* start, int side, bool two_sided, int d) {
  const int n = two_sided ? abs(d) : -d;
  int b = 0;  // the last bucket that starts at n or below (start[0] is 0; what lies behind `side` starts nowhere), and 0 ahead of a one-sided bias
#pragma unroll
  for (int step = kMaxSide / 2; step > 0; step >>= 1) b += start[b + step] <= n ? step : 0;
  return d > 0 && two_sided ? side + b : side - 1 - b;
}
RA_DEV int table_row(int ordered, int side) { return ordered >= side ? ordered : side - 1 - ordered; }
// N: the distances of a tile
template <int N, bool GRAD>
struct BiasLds {
  static_assert(N <= 256, "first");
  float value[2][N];          // of the tiles of the two buffers
  float table[2 * kMaxSide];  // of this head, in the order of d
  int start[kMaxSide];
  int lo[GRAD ? 2 * kMaxSide : 1], hi[GRAD ? 2 * kMaxSide : 1];  // the distances of a bucket (in that order; hi < lo: none)
  unsigned char first[2][GRAD ? N : 1];  // where the bucket of a tile's distance begins among them
};
RA_DEV float load_table(const TermArgs& t, int row, int h) {
  const long long at = row * t.table_sb + h * t.table_sh;
  if (t.table_dtype == RA_DTYPE_F32) return ((const float*)t.table)[at];
  if (t.table_dtype == RA_DTYPE_F16) return (float)((const _Float16*)t.table)[at];
  return (float)((const bf16_t*)t.table)[at];
}
// What a wave knows about the bias: from where on it is constant, and what it is there (times log2(e), for an exponent).
struct BiasEnds {
  int far, future;    // d <= -far, d >= future
  float past, ahead;
};
template <int N, bool GRAD>
RA_DEV BiasEnds load_bias(const TermArgs& t, int h, float unit, BiasLds<N, GRAD>& lds) {
  const int tid = threadIdx.x, n = t.two_sided ? 2 * t.side : t.side;
  if constexpr (GRAD) {
    if (tid < 2 * kMaxSide) {
      constexpr int kFar = 1 << 30;
      const bool ahead = tid >= t.side;
      const int b = ahead ? tid - t.side : t.side - 1 - tid;
      int lo = 0, hi = -1;
      if (tid < n) {
        const int from = t.start[b], to = b + 1 < t.side ? t.start[b + 1] - 1 : kFar;  // |d|
        lo = ahead ? max(from, 1) : -to;
        hi = ahead ? to : b == 0 && !t.two_sided ? kFar : -from;
      }
      lds.lo[tid] = lo;
      lds.hi[tid] = hi;
    }
  }
  if (tid < n) lds.table[tid] = load_table(t, table_row(tid, t.side), h) * unit;
  if (tid < kMaxSide) lds.start[tid] = tid < t.side ? t.start[tid] : 0x7fffffff;
  BiasEnds e;
  e.far = t.start[t.side - 1];
  e.future = t.two_sided ? e.far : t.start[1] > 0 ? 0 : 1;  // (distance 0 itself may lie in a later bucket than the keys ahead)
  auto uniform = [](float x) {  // (the product, not its factor: a scalar register has no product of its own, and the backward no vector register for it)
    asm volatile("" : "+v"(x));
    return __uint_as_float((unsigned)__builtin_amdgcn_readfirstlane((int)__float_as_uint(x)));
  };
  e.past = uniform(load_table(t, t.side - 1, h) * kLog2e);
  e.ahead = uniform(load_table(t, t.two_sided ? 2 * t.side - 1 : 0, h) * kLog2e);
  return e;
}
// The values of the distances d_lo .. d_lo + N - 1 of a tile for the buffer `buf`; all threads of the workgroup.
template <int N, bool GRAD>
RA_DEV void write_bias(const TermArgs& t, const BiasEnds& e, BiasLds<N, GRAD>& lds, int buf, int d_lo) {
  if (d_lo + N - 1 <= -e.far || d_lo >= e.future) return;  // constant: nothing reads it
  int i = threadIdx.x;
  asm volatile("" : "+v"(i));  // (addresses made here: one that is kept may be spilled, and its reload waits for the tile's loads)
  if (i < N) {
    const int u = ordered_bucket(lds.start, t.side, t.two_sided, d_lo + i);
    lds.value[buf][i] = lds.table[u];
    if constexpr (GRAD) lds.first[buf][i] = (unsigned char)max(lds.lo[u] - d_lo, 0);
  }
}

// What four elements of the output lack of their value once they are rounded to T, rounded itself.
template <typename T>
RA_DEV void store_rest(void* base, long long at, const f32x4& x) {
  f32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = x[e] - (float)(T)x[e];
  store_as<T>(base, at, r);
}

// Sum over a wave, in every lane.
RA_DEV float wave_sum(float x) {
  x += __uint_as_float(lane_dpp<0xb1>(__float_as_uint(x)));
  x += __uint_as_float(lane_dpp<0x4e>(__float_as_uint(x)));
  x += __uint_as_float(lane_dpp<0x141>(__float_as_uint(x)));
  x += __uint_as_float(lane_dpp<0x140>(__float_as_uint(x)));
  auto lane = [&](int l) { return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(x), l)); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// Sums of a wave's lanes from lane `first` (each lane's own, the same for all lanes on the way to it) up to and including each.  A sum takes nothing from
// lanes before its first one, not even to subtract it again.
RA_DEV float wave_scan(float x, int lane, int first) {
  auto add = [&](auto ctrl, auto rows, bool same) {
    const float y = __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    x += same ? y : 0.f;
  };
  using All = std::integral_constant<int, 0xf>;
  add(std::integral_constant<int, 0x111>{}, All{}, lane - 1 >= first);  // one lane to the right inside rows of 16, two, four, eight
  add(std::integral_constant<int, 0x112>{}, All{}, lane - 2 >= first);
  add(std::integral_constant<int, 0x114>{}, All{}, lane - 4 >= first);
  add(std::integral_constant<int, 0x118>{}, All{}, lane - 8 >= first);
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}, (lane & 48) > first);  // the last lane of a row to the next row, of the first half to the second
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}, 32 > first);
  return x;
}
// lane (from / 4) mod 64's value
RA_DEV float lane_at(int from, float x) { return __uint_as_float((unsigned)__builtin_amdgcn_ds_bpermute(from, (int)__float_as_uint(x))); }

}  // namespace ra
