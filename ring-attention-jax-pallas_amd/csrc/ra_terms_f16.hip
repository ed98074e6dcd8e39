// The pair kernels with a relative bias or dropout on operands in fp16.
#include "ra_terms_launch.h"

namespace ra {

hipError_t launch_fwd_f16(const PairFwdTermArgs& a, int D, hipStream_t stream) { return launch_fwd<6>(a, D, stream); }
hipError_t launch_bwd_f16(const PairBwdArgs& dkdv, const PairBwdArgs& dq, const TermArgs& t, int D, hipStream_t stream) {
  return launch_bwd<6>(dkdv, dq, t, D, stream);
}
hipError_t launch_stat_f16(const StatArgs& a, int out_f32, int dout_dtype, int D, hipStream_t stream) {
  return launch_stat<_Float16>(a, out_f32, dout_dtype, D, stream);
}

}  // namespace ra
