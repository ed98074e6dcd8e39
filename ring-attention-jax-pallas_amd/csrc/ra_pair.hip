// Launches of the kernels of ra_pair_kernels.h.
#include "ra_pair_kernels.h"

namespace ra {

template <int D>
static hipError_t launch_pair_sum_d(const PairBwdArgs* dkdv, const PairBwdArgs* dq, hipStream_t stream) {
  const bool sum_dkdv = dkdv && dkdv->n_split > 1, sum_dq = dq && dq->n_split > 1;
  if (!(sum_dkdv || sum_dq)) return hipSuccess;
  const PairBwdArgs& any = dkdv ? *dkdv : *dq;
  const long long n = (long long)any.a.B * any.a.H * std::max(sum_dkdv ? any.a.Lk : 0, sum_dq ? any.a.Lq : 0) * (D / 4);
  const BothBwdArgs p{sum_dkdv ? *dkdv : *dq, sum_dq ? *dq : *dkdv, 0, 0};
  hipLaunchKernelGGL((pair_sum_kernel<D>), dim3((unsigned)((n + 255) / 256), (unsigned)(2 * sum_dkdv + sum_dq)), dim3(kPairThreads), 0, stream, p,
                     sum_dkdv ? 0 : 2);
  return hipGetLastError();
}
hipError_t launch_pair_sum(const PairBwdArgs* dkdv, const PairBwdArgs* dq, int D, hipStream_t stream) {
  return with_dim(D, 0, [&](auto d) { return launch_pair_sum_d<d.value>(dkdv, dq, stream); });
}

// dkdv, dq: nullptr for none
template <int D, int MODE>
static hipError_t launch_bwd_pair_dm(const PairBwdArgs* dkdv, const PairBwdArgs* dq, hipStream_t stream) {
  auto tiles = [](int L) { return (L + kPairRows - 1) / kPairRows; };
  const int n_dkdv = dkdv ? dkdv->a.B * dkdv->a.H * dkdv->n_split * tiles(dkdv->a.Lk) : 0;
  const int n_dq = dq ? dq->a.B * dq->a.H * dq->n_split * tiles(dq->a.Lq) : 0;
  const dim3 block(kPairThreads);
  if (dkdv && dq) {
    const bool dq_first = dq->chunk_tiles > dkdv->chunk_tiles;
    const BothBwdArgs p{*dkdv, *dq, dq_first ? n_dq : n_dkdv, dq_first};
    hipLaunchKernelGGL((bwd_pair_kernel<D, MODE>), dim3((unsigned)(n_dkdv + n_dq)), block, 0, stream, p);
  } else if (dkdv) {
    hipLaunchKernelGGL((dkdv_pair_kernel<D, MODE>), dim3((unsigned)n_dkdv), block, 0, stream, *dkdv);
  } else {
    hipLaunchKernelGGL((dq_pair_kernel<D, MODE>), dim3((unsigned)n_dq), block, 0, stream, *dq);
  }
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? launch_pair_sum_d<D>(dkdv, dq, stream) : e;
}

hipError_t launch_bwd_pair(const PairBwdArgs* dkdv, const PairBwdArgs* dq, int D, int mode, hipStream_t stream) {
  return with_dim(D, mode, [&](auto d) {
    if (mode == 2) {
      if constexpr (d.value == 64 || d.value == 128) return launch_bwd_pair_dm<d.value, 2>(dkdv, dq, stream);
    }
    return mode == 1 ? launch_bwd_pair_dm<d.value, 1>(dkdv, dq, stream) : launch_bwd_pair_dm<d.value, 0>(dkdv, dq, stream);
  });
}

hipError_t launch_pair_stat(const StatArgs& a, int out_f32, int dout_dtype, int D, hipStream_t stream) {
  return with_dim(D, 0, [&](auto d) {
    auto with_out = [&](auto out) {
      using OutT = decltype(out);
      if (dout_dtype == RA_DTYPE_F32) return launch_pair_stat_d<OutT, float, bf16_t, false, d.value>(a, stream);
      if (dout_dtype == RA_DTYPE_F16) return launch_pair_stat_d<OutT, _Float16, bf16_t, false, d.value>(a, stream);
      return launch_pair_stat_d<OutT, bf16_t, bf16_t, false, d.value>(a, stream);
    };
    return out_f32 ? with_out(float{}) : with_out(bf16_t{});
  });
}

template <int D>
static hipError_t launch_fwd_pair_d(const PairFwdArgs& a, int mode, hipStream_t stream) {
  const int nqt = (a.Lq + kPairRows - 1) / kPairRows;
  dim3 grid((unsigned)(a.B * a.H * a.n_split * nqt)), block(kPairThreads);
  if (mode == 2) {
    if constexpr (D == 64 || D == 128) hipLaunchKernelGGL((fwd_pair_kernel<D, 2>), grid, block, 0, stream, a);
  } else if (mode == 1) {
    hipLaunchKernelGGL((fwd_pair_kernel<D, 1>), grid, block, 0, stream, a);
  } else {
    hipLaunchKernelGGL((fwd_pair_kernel<D, 0>), grid, block, 0, stream, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.part_o == nullptr) return e;
  return launch_pair_combine<D, 0>(a, stream);
}

hipError_t launch_fwd_pair(const PairFwdArgs& a, int D, int mode, hipStream_t stream) {
  return with_dim(D, mode, [&](auto d) { return launch_fwd_pair_d<d.value>(a, mode, stream); });
}

}  // namespace ra
