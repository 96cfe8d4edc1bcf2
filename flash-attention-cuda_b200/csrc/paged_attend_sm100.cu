// Attention of new tokens over a paged K/V cache (fa_attend_paged).
//
//   o_i = sum_j exp(scale q_i k_j - m_i) v_j / l_i,  j over the rows that
//   token i sees, m_i and l_i the running maximum and sum.
//
// One warp per (token, head): lanes share the head's elements, keys one by
// one, the softmax running.

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fa_kernels.h"
#include "fa_sm100.cuh"

namespace fa {
namespace paged {

constexpr int kThreads = 128;

template <typename Dt, int D>
__global__ void __launch_bounds__(kThreads) attend_paged_kernel(const PagedArgs a) {
  const int lane = threadIdx.x & 31;
  const long long w =
      (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int t = static_cast<int>(w / a.H);
  const int h = static_cast<int>(w % a.H);
  if (t >= a.tokens) return;
  int seq = 0;
  for (int b = lane; b < a.batch; b += 32) seq += a.starts[b + 1] <= t;
  seq = __reduce_add_sync(0xffffffffu, seq);
  if (seq >= a.batch) return;
  const long long len = a.seq_lens[seq];
  const long long row = len - a.starts[seq + 1] + t;
  long long n = a.causal ? row + 1 : len;
  n = min(n, static_cast<long long>(a.table_width) * a.page_rows);
  const int kv = h / (a.H / a.H_kv);

  constexpr int E = D / 32;
  float q[E], o[E];
  const __half *qp = a.q + t * a.q_st + h * a.q_sh;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = Dt::unpack2(__half_as_ushort(qp[lane + 32 * i])).x * a.scale_log2;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (long long j = 0; j < n; ++j) {
    const int page = a.page_table[seq * a.table_stride + j / a.page_rows];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) record_error(FA_ERR_PAGE);
      break;
    }
    const long long r = j % a.page_rows;
    const __half *kp = a.k_pages + page * a.kp_sp + kv * a.kp_sh + r * a.kp_sr;
    const __half *vp = a.v_pages + page * a.vp_sp + kv * a.vp_sh + r * a.vp_sr;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i)
      x = fmaf(q[i], Dt::unpack2(__half_as_ushort(kp[lane + 32 * i])).x, x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
    const float mn = fmaxf(m, x);
    const float corr = exp2f(m - mn);
    const float p = exp2f(x - mn);
    m = mn;
    l = fmaf(l, corr, p);
#pragma unroll
    for (int i = 0; i < E; ++i)
      o[i] = fmaf(o[i], corr,
                  p * Dt::unpack2(__half_as_ushort(vp[lane + 32 * i])).x);
  }
  __half *op = a.out + (static_cast<long long>(t) * a.H + h) * D;
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i)
    op[lane + 32 * i] = store_elem(o[i] * inv, Dt::kDtype);
  if (a.lse && lane == 0)
    a.lse[static_cast<long long>(t) * a.H + h] =
        l > 0.f ? 0.69314718055994531f * (m + log2f(l)) : -INFINITY;
}

}  // namespace paged

size_t attend_paged_workspace_bytes(int, int) { return 16; }

cudaError_t launch_attend_paged_kernel(const PagedArgs &a, int dtype,
                                       cudaStream_t stream) {
  const long long warps = static_cast<long long>(a.tokens) * a.H;
  const unsigned grid =
      static_cast<unsigned>((warps * 32 + paged::kThreads - 1) / paged::kThreads);
  auto kernel =
      dtype == FA_DTYPE_BF16
          ? (a.D == 64 ? paged::attend_paged_kernel<BF16, 64>
                       : paged::attend_paged_kernel<BF16, 128>)
          : (a.D == 64 ? paged::attend_paged_kernel<F16, 64>
                       : paged::attend_paged_kernel<F16, 128>);
  kernel<<<grid, paged::kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace fa
