// key_weights.cu - the attention each prompt key received:
//   w_j = sum over queries i in [max(j, first), L) of 2^(x_ij - lse_i),
//   x_ij = log2e (q_i.k_j / 8 + lam_h exp(min(g_i - g_j, 0)) (c_i.b~_j) + (F_i - F_j)),
// with lse from the attention forward. Every key is owned by one thread, which adds its queries in
// order: no atomics.
#include <cuda_runtime.h>
#include <cstdint>

#include "sm100.cuh"
#include "key_weights.h"

namespace sisa {
namespace kwt {

constexpr int NT = 128, QT = 32;
constexpr float kLog2e = 1.4426950408889634f;

template <bool kHalf>
__global__ void __launch_bounds__(NT) key_weights_kernel(KeyWeightParams p) {
  __shared__ float s_q[QT][64], s_c[QT][32], s_g[QT], s_a[QT];
  const int bh = blockIdx.y, b = bh / p.H, h = bh % p.H, tid = threadIdx.x;
  const int k0 = blockIdx.x * NT, j = k0 + tid;
  const bool ok = j < p.L;
  float kr[64], br[32];
  const uint4* kp = reinterpret_cast<const uint4*>(p.k + 2 * (b * p.k_sb + h * p.k_sh + (int64_t)(ok ? j : 0) * p.k_sl));
  const uint4* bp = reinterpret_cast<const uint4*>(p.b + 2 * (b * p.b_sb + h * p.b_sh + (int64_t)(ok ? j : 0) * p.b_sl));
#pragma unroll
  for (int i = 0; i < 12; ++i) {
    const uint4 v = i < 8 ? kp[i] : bp[i - 8];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float* d = i < 8 ? kr + 8 * i : br + 8 * (i - 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) { d[2 * e] = unpack_lo<kHalf>(w[e]); d[2 * e + 1] = unpack_hi<kHalf>(w[e]); }
  }
  const float* pos = p.pos + (int64_t)bh * 4 * p.Lp;
  const float gj = ok ? pos[j] : 0.f, fj = ok ? pos[p.Lp + j] : 0.f;
  const float lam = p.lam[h];
  float acc = 0.f;
  for (int i0 = max(p.first, k0) / QT * QT; i0 < p.L; i0 += QT) {
    __syncthreads();
    for (int e = tid; e < QT * 96; e += NT) {
      const int r = e / 96, d = e % 96, i = i0 + r;
      float x = 0.f;
      if (i < p.L) {
        const char* src = d < 64 ? p.q + 2 * (b * p.q_sb + h * p.q_sh + i * p.q_sl + d)
                                 : p.c + 2 * (b * p.c_sb + h * p.c_sh + i * p.c_sl + d - 64);
        x = unpack_lo<kHalf>(*reinterpret_cast<const uint16_t*>(src));
      }
      if (d < 64) s_q[r][d] = x; else s_c[r][d - 64] = x;
    }
    if (tid < QT && i0 + tid < p.L) {
      s_g[tid] = pos[i0 + tid];
      s_a[tid] = p.lse[(int64_t)bh * p.L + i0 + tid];
    }
    __syncthreads();
    const int hi = min(QT, p.L - i0);
    for (int r = 0; r < hi; ++r) {
      const int i = i0 + r;
      if (!ok || i < j || i < p.first) continue;
      float qk = 0.f, cb = 0.f;
#pragma unroll
      for (int d = 0; d < 64; ++d) qk = fmaf(s_q[r][d], kr[d], qk);
#pragma unroll
      for (int d = 0; d < 32; ++d) cb = fmaf(s_c[r][d], br[d], cb);
      const float dec = exp2f(fmin_nan((s_g[r] - gj) * kLog2e, 0.f));
      const float s = fmaf(qk, 0.125f, lam * (dec * cb)) + (pos[p.Lp + i] - fj);
      acc += exp2f(fmaf(s, kLog2e, -s_a[r]));
    }
  }
  if (ok) p.w[(int64_t)bh * p.L + j] = acc;
  if (ok && !isfinite(acc) && p.status) atomicOr(p.status, SISA_ST_NONFINITE);
}

}  // namespace kwt

cudaError_t launch_key_weights(const KeyWeightParams& p, int dtype, cudaStream_t st) {
  dim3 grid((p.L + kwt::NT - 1) / kwt::NT, p.B * p.H);
  if (dtype == 1) kwt::key_weights_kernel<true><<<grid, kwt::NT, 0, st>>>(p);
  else kwt::key_weights_kernel<false><<<grid, kwt::NT, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace sisa
