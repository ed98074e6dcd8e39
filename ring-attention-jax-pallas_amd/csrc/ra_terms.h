// Device code of the terms that take arguments of their own (TermArgs): the relative position bias by buckets, and dropout.
#pragma once
#include "ra_launch.h"

namespace ra {

// ------------------------------------------------------------------------------------------------
// Dropout.  A weight (query i, key j) of head hh (batch * heads + head) has 16 bits of a counter-based generator: Philox 4x32 of seven rounds
// (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011: the fewest that pass all of their tests) with the
// seed as key and the counter (j / 2, i / 4, hh, 0); query i's word is the (i % 4)-th, an even key's half the low one.  A call serves eight weights
// whichever side the kernel's lanes own: four neighbouring lanes with a query each exchange words, and two with a key each halves.
// ------------------------------------------------------------------------------------------------
struct Philox {
  unsigned c0, c1, c2, c3;
  RA_DEV void start(unsigned k_pair, unsigned q_group, unsigned hh) {
    c0 = k_pair;
    c1 = q_group;
    c2 = hh;
    c3 = 0;
  }
  // rounds [FROM, TO) under the key k0, k1
  template <int FROM, int TO>
  RA_DEV void rounds(unsigned k0, unsigned k1) {
#pragma unroll
    for (int r = FROM; r < TO; ++r) {
      const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
      const unsigned x0 = k0 + (unsigned)r * 0x9E3779B9u, x1 = k1 + (unsigned)r * 0xBB67AE85u;
      c0 = (unsigned)(b >> 32) ^ c1 ^ x0;
      c1 = (unsigned)b;
      c2 = (unsigned)(a >> 32) ^ c3 ^ x1;
      c3 = (unsigned)a;
    }
  }
};
constexpr int kPhiloxRounds = 7;

template <int CTRL>
RA_DEV unsigned quad_dpp(unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
// The words w0 .. w3 of four neighbouring lanes turned round: word x of a lane becomes the lane's own word of lane x.
RA_DEV void quad_transpose(unsigned (&w)[4], int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
#pragma unroll
  for (int x = 0; x < 4; x += 2) {
    const unsigned got = quad_dpp<0xb1>(b0 ? w[x] : w[x + 1]);
    w[x] = b0 ? got : w[x];
    w[x + 1] = b0 ? w[x + 1] : got;
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const unsigned got = quad_dpp<0x4e>(b1 ? w[x] : w[x + 2]);
    w[x] = b1 ? got : w[x];
    w[x + 2] = b1 ? w[x + 2] : got;
  }
}
// Whether the weight of a word's half stays.
RA_DEV bool stays_low(unsigned w, unsigned drop) { return (unsigned short)w >= (unsigned short)drop; }
RA_DEV bool stays_high(unsigned w, unsigned drop) { return w >= drop << 16; }

// The seed's words, as uniform values.
RA_DEV void load_seed(const TermArgs& t, unsigned& k0, unsigned& k1) {
  const unsigned long long s = t.seed_at != nullptr ? *t.seed_at : t.seed;
  k0 = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)s);
  k1 = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(s >> 32));
}

// ------------------------------------------------------------------------------------------------
// The relative bias.  It is a function of the distance d = key - query, constant from the last bucket's start on (and, one-sided, from 0 on): a
// block of 32 x 32 scores that lies there takes one number into its exponents, and no other work.  For the tiles on the way the
// workgroup writes the values of a tile's distances to LDS, one a thread, while the tile is on its way, and a score reads its own.
// ------------------------------------------------------------------------------------------------
// Buckets in the order of d: the far past first, the far future last (one-sided: bucket 0 last).
RA_DEV int ordered_bucket(const int* start, int side, bool two_sided, int d) {
  const int n = two_sided ? abs(d) : max(-d, 0);
  int b = 0;  // the last bucket that starts at n or below (start[0] is 0; what lies behind `side` starts nowhere)
#pragma unroll
  for (int step = kMaxSide / 2; step > 0; step >>= 1) b += start[b + step] <= n ? step : 0;
  return d > 0 && two_sided ? side + b : side - 1 - b;
}
RA_DEV int table_row(int ordered, int side) { return ordered >= side ? ordered : side - 1 - ordered; }
// N: the distances of a tile
template <int N, bool GRAD>
struct BiasLds {
  float value[2][N];             // of the tiles of the two buffers
  unsigned char ordered[GRAD ? 2 : 1][GRAD ? N : 4];  // their buckets
  float table[2 * kMaxSide];     // of this head, in the order of d
  int start[kMaxSide];
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
template <typename Lds>
RA_DEV BiasEnds load_bias(const TermArgs& t, int h, float unit, Lds& lds) {
  const int tid = threadIdx.x, n = t.two_sided ? 2 * t.side : t.side;
  if (tid < n) lds.table[tid] = load_table(t, table_row(tid, t.side), h) * unit;
  if (tid < kMaxSide) lds.start[tid] = tid < t.side ? t.start[tid] : 0x7fffffff;
  BiasEnds e;
  e.far = t.start[t.side - 1];
  e.future = t.two_sided ? e.far : 0;
  e.past = load_table(t, t.side - 1, h) * kLog2e;
  e.ahead = load_table(t, t.two_sided ? 2 * t.side - 1 : 0, h) * kLog2e;
  e.past = __uint_as_float((unsigned)__builtin_amdgcn_readfirstlane((int)__float_as_uint(e.past)));
  e.ahead = __uint_as_float((unsigned)__builtin_amdgcn_readfirstlane((int)__float_as_uint(e.ahead)));
  return e;
}
// The values of the distances d_lo .. d_lo + N - 1 of a tile for the buffer `buf`; all threads of the workgroup.
template <int N, bool GRAD>
RA_DEV void write_bias(const TermArgs& t, const BiasEnds& e, BiasLds<N, GRAD>& lds, int buf, int d_lo) {
  if (d_lo + N - 1 <= -e.far || d_lo >= e.future) return;  // constant: nothing reads it
  const int i = threadIdx.x;
  if (i < N) {
    const int u = ordered_bucket(lds.start, t.side, t.two_sided, d_lo + i);
    lds.value[buf][i] = lds.table[u];
    if constexpr (GRAD) lds.ordered[buf][i] = (unsigned char)u;
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
  x += __uint_as_float(quad_dpp<0xb1>(__float_as_uint(x)));
  x += __uint_as_float(quad_dpp<0x4e>(__float_as_uint(x)));
  x += __uint_as_float(quad_dpp<0x141>(__float_as_uint(x)));
  x += __uint_as_float(quad_dpp<0x140>(__float_as_uint(x)));
  auto lane = [&](int l) { return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(x), l)); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

}  // namespace ra
