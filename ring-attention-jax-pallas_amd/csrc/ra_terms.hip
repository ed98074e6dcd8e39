// The pair kernels with the terms that take arguments of their own, the relative bias and dropout, and the sum of the bias's gradient.
#include "ra_terms_launch.h"

namespace ra {

// The relative bias's gradient from the workgroups' sums: a workgroup per head, a thread per bucket and row in turn, always in the same order.
// Bound by latency: the sums come from all over the chip.  Eight rows a thread are on their way at once (one after the other: 9.2 us at 2 x 32 tiles, 32
// buckets, H=16; now 5.2, of which the 0.5 MB would be 0.1 at a large copy's rate).
constexpr int kGradThreads = 512, kGradAhead = 8;
__global__ __launch_bounds__(kGradThreads) void table_grad_kernel(const TermArgs t, const int* part_n, int B, int H, int tiles, int n_split) {
  __shared__ float s_sum[kGradThreads];
  const int n = t.two_sided ? 2 * t.side : t.side, h = blockIdx.x, tid = threadIdx.x;
  int width = 2;
  while (width < n) width *= 2;
  const int u = tid % width, first = tid / width, step = kGradThreads / width;
  float sum = 0.f;
  const int rows = B * tiles * n_split;
  for (int i0 = first; i0 < rows; i0 += kGradAhead * step) {
    float x[kGradAhead];
    int pieces[kGradAhead];
#pragma unroll
    for (int a = 0; a < kGradAhead; ++a) {
      const int i = min(i0 + a * step, rows - 1), tile = i / n_split % tiles, b = i / n_split / tiles;
      const long long at = ((long long)b * H + h) * tiles + tile;
      const float* row = t.grad_part + (at * n_split + i % n_split) * kGradRow;
      pieces[a] = part_n != nullptr ? max(part_n[at], 1) : 1;
      x[a] = row[min(u, n - 1)];  // (of a share that there is not: whatever lies there)
    }
#pragma unroll
    for (int a = 0; a < kGradAhead; ++a) {
      const int i = i0 + a * step;
      sum += i < rows && i % n_split < pieces[a] ? x[a] : 0.f;
    }
  }
  s_sum[tid] = sum;
  __syncthreads();
  if (tid >= n) return;
  for (int i = 1; i < step; ++i) sum += s_sum[tid + i * width];
  const long long at = (long long)table_row(tid, t.side) * H + h;
  if (t.table_dtype == RA_DTYPE_F32) ((float*)t.grad)[at] = sum;
  else if (t.table_dtype == RA_DTYPE_F16) ((_Float16*)t.grad)[at] = (_Float16)sum;
  else ((bf16_t*)t.grad)[at] = (bf16_t)sum;
}

hipError_t launch_fwd_terms(const PairFwdTermArgs& a, int D, hipStream_t stream) {
  return a.t.half ? launch_fwd_f16(a, D, stream) : launch_fwd<3>(a, D, stream);
}

hipError_t launch_terms_stat(const StatArgs& a, bool half, int out_f32, int dout_dtype, int D, hipStream_t stream) {
  return half ? launch_stat_f16(a, out_f32, dout_dtype, D, stream) : launch_stat<bf16_t>(a, out_f32, dout_dtype, D, stream);
}

hipError_t launch_bwd_terms(const PairBwdArgs& dkdv, const PairBwdArgs& dq, const TermArgs& t, int D, hipStream_t stream) {
  hipError_t e = t.half ? launch_bwd_f16(dkdv, dq, t, D, stream) : launch_bwd<3>(dkdv, dq, t, D, stream);
  if (e != hipSuccess || (e = launch_pair_sum(&dkdv, &dq, D, stream)) != hipSuccess || t.grad_part == nullptr) return e;
  const int tiles = (dq.a.Lq + kPairRows - 1) / kPairRows;
  hipLaunchKernelGGL(table_grad_kernel, dim3((unsigned)dq.a.H), dim3(kGradThreads), 0, stream, t, dq.part_n, dq.a.B, dq.a.H, tiles, dq.n_split);
  return hipGetLastError();
}

}  // namespace ra
