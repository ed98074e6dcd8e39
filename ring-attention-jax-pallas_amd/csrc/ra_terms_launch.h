// The launches of one element type: FIRST is the mode with the relative bias alone.
#pragma once
#include "ra_pair_kernels.h"

namespace ra {

template <int FIRST, typename Launch>
static hipError_t with_terms(int D, const TermArgs& t, Launch launch) {
  return with_dim(D, FIRST, [&](auto d) {
    if (t.table == nullptr) return launch(d, std::integral_constant<int, FIRST + 1>{});
    if (t.drop == 0) return launch(d, std::integral_constant<int, FIRST>{});
    return launch(d, std::integral_constant<int, FIRST + 2>{});
  });
}

template <int FIRST>
static hipError_t launch_fwd(const PairFwdTermArgs& a, int D, hipStream_t stream) {
  const int nqt = (a.Lq + kPairRows - 1) / kPairRows;
  const dim3 grid((unsigned)(a.B * a.H * a.n_split * nqt)), block(kPairThreads);
  return with_terms<FIRST>(D, a.t, [&](auto d, auto mode) {
    hipLaunchKernelGGL((fwd_pair_kernel<d.value, mode.value>), grid, block, 0, stream, a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || a.part_o == nullptr ? e : launch_pair_combine<d.value, FIRST>(a, stream);
  });
}

template <int FIRST>
static hipError_t launch_bwd(const PairBwdArgs& dkdv, const PairBwdArgs& dq, const TermArgs& t, int D, hipStream_t stream) {
  auto tiles = [](int L) { return (L + kPairRows - 1) / kPairRows; };
  const int n_dkdv = dkdv.a.B * dkdv.a.H * dkdv.n_split * tiles(dkdv.a.Lk), n_dq = dq.a.B * dq.a.H * dq.n_split * tiles(dq.a.Lq);
  BothTermArgs p;
  p.dkdv = dkdv;
  p.dq = dq;
  p.dq_first = dq.chunk_tiles > dkdv.chunk_tiles;
  p.n_first = p.dq_first ? n_dq : n_dkdv;
  p.t = t;
  return with_terms<FIRST>(D, t, [&](auto d, auto mode) {
    hipLaunchKernelGGL((bwd_pair_kernel<d.value, mode.value>), dim3((unsigned)(n_dkdv + n_dq)), dim3(kPairThreads), 0, stream, p);
    return hipGetLastError();
  });
}

template <typename T>
static hipError_t launch_stat(const StatArgs& a, int out_f32, int dout_dtype, int D, hipStream_t stream) {
  return with_dim(D, 0, [&](auto d) {
    auto with_out = [&](auto out, auto rest) {
      using OutT = decltype(out);
      if (dout_dtype == RA_DTYPE_F32) return launch_pair_stat_d<OutT, float, T, rest.value, d.value>(a, stream);
      if (dout_dtype == RA_DTYPE_F16) return launch_pair_stat_d<OutT, _Float16, T, rest.value, d.value>(a, stream);
      return launch_pair_stat_d<OutT, bf16_t, T, rest.value, d.value>(a, stream);
    };
    if (a.rest != nullptr) return with_out(T{}, std::true_type{});
    return out_f32 ? with_out(float{}, std::false_type{}) : with_out(T{}, std::false_type{});
  });
}

// (ra_terms_f16.hip)
hipError_t launch_fwd_f16(const PairFwdTermArgs& a, int D, hipStream_t stream);
hipError_t launch_bwd_f16(const PairBwdArgs& dkdv, const PairBwdArgs& dq, const TermArgs& t, int D, hipStream_t stream);
hipError_t launch_stat_f16(const StatArgs& a, int out_f32, int dout_dtype, int D, hipStream_t stream);

}  // namespace ra
