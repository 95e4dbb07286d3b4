// paged_attn.cu - attention of one new token per sequence over its paged keys.
//
// For every sequence b with n_b keys (slots 0 .. n_b - 1 of its pages, in any order) and head h:
//   x_j = log2e (q.k_j / 8 + lam_h exp(min(g_q - g_j, 0)) (c.b~_j) + (F_q - F_j)),
//   y = sum_j 2^(x_j - lse) v_j,  lse = log2 sum_j 2^x_j,  and optionally weight_j += 2^(x_j - lse).
// A row with no keys gives y = 0 and lse = -inf.
#include <cuda_runtime.h>
#include <cstdint>

#include "sm100.cuh"
#include "paged.h"

namespace sisa {
namespace pat {

constexpr int NT = 256, NW = NT / 32;
constexpr float kLog2e = 1.4426950408889634f;

template <bool kHalf>
__device__ __forceinline__ void unpack8(const uint4& v, float* out) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    out[2 * e] = unpack_lo<kHalf>(w[e]);
    out[2 * e + 1] = unpack_hi<kHalf>(w[e]);
  }
}

__device__ __forceinline__ int64_t keys_of(const PagedAttnParams& p, int b) {
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : (n > p.max_keys ? p.max_keys : n);
}

// Grid (splits, B*H). Eight lanes per key, each with 16 bytes of the key's k, v and b~ rows; every warp
// runs its own online softmax over groups of four keys, merged once at the end.
template <bool kHalf>
__global__ void __launch_bounds__(NT) paged_split_kernel(PagedAttnParams p) {
  const int split = blockIdx.x, bh = blockIdx.y;
  const int b = bh / p.H, h = bh % p.H;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t N = keys_of(p, b);
  if (split == 0 && h == 0 && tid == 0 && p.lengths[b] > p.max_keys && p.status) atomicOr(p.status, SISA_ST_BAD_POS);
  const int64_t per = (N + p.splits - 1) / p.splits;
  const int64_t j_begin = split * per, j_end = min(N, j_begin + per);
  __shared__ float s_m[NW], s_l[NW];
  __shared__ float s_acc[NW][64];
  const int sub = lane >> 3, part = lane & 7;
  float q8[8], c8[8];
  unpack8<kHalf>(reinterpret_cast<const uint4*>(p.q + 2 * ((int64_t)b * p.q_sb + (int64_t)h * p.q_sh))[part], q8);
  uint4 cv = make_uint4(0, 0, 0, 0);
  if (part < 4) cv = reinterpret_cast<const uint4*>(p.c + 2 * ((int64_t)b * p.c_sb + (int64_t)h * p.c_sh))[part];
  unpack8<kHalf>(cv, c8);
  const float gq = p.g_q[bh], fq = p.f_q ? p.f_q[bh] : 0.f;
  const float c1 = 0.125f * kLog2e, lam2 = p.lam[h] * kLog2e;
  float* xs = p.weight_out ? p.ws + (int64_t)p.splits * p.B * p.H * 66 + (int64_t)bh * p.max_keys : nullptr;
  float m_ref = -INFINITY, lsum = 0.f, acc[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) acc[d] = 0.f;
#pragma unroll 1
  for (int64_t j0 = j_begin + 4 * warp; j0 < j_end; j0 += 4 * NW) {
    const int64_t j = j0 + sub;
    const int page = j < j_end ? page_of(p.pg, b, j, p.status) : -1;
    const bool ok = page >= 0;
    uint4 kv = make_uint4(0, 0, 0, 0), vv = kv, bv = kv;
    float gj = 0.f, fj = 0.f;
    if (ok) {
      const int64_t slot = j & ((1 << p.pg.page_shift) - 1);
      kv = reinterpret_cast<const uint4*>(p.pg.k + 2 * (page * p.pg.k_sp + h * p.pg.k_sh + slot * 64))[part];
      vv = reinterpret_cast<const uint4*>(p.pg.v + 2 * (page * p.pg.v_sp + h * p.pg.v_sh + slot * 64))[part];
      if (part < 4) bv = reinterpret_cast<const uint4*>(p.pg.b + 2 * (page * p.pg.b_sp + h * p.pg.b_sh + slot * 32))[part];
      gj = p.pg.g[page * p.pg.s_sp + h * p.pg.s_sh + slot];
      if (p.f_q) fj = p.pg.f[page * p.pg.s_sp + h * p.pg.s_sh + slot];
    }
    float k8[8], b8[8], v8[8];
    unpack8<kHalf>(kv, k8);
    unpack8<kHalf>(bv, b8);
    unpack8<kHalf>(vv, v8);
    float qk = 0.f, cb = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qk = fmaf(q8[e], k8[e], qk);
      cb = fmaf(c8[e], b8[e], cb);
    }
    const float dec = exp2f(fmin_nan((gq - gj) * kLog2e, 0.f));
    float x = fmaf(qk, c1, lam2 * (dec * cb));
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    x += __shfl_xor_sync(0xffffffffu, x, 4);
    x = ok ? fmaf(fq - fj, kLog2e, x) : -INFINITY;
    if (xs && part == 0 && j < j_end) xs[j] = x;
    float mx = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
    if (mx > m_ref + 8.f) {
      const float corr = (m_ref == -INFINITY) ? 0.f : exp2f(m_ref - mx);
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[d] *= corr;
      lsum *= corr;
      m_ref = mx;
    }
    const float pj = ok ? exp2f(x - (m_ref == -INFINITY ? 0.f : m_ref)) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(pj, v8[e], acc[e]);
    lsum += pj;
  }
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    acc[d] += __shfl_xor_sync(0xffffffffu, acc[d], 8);
    acc[d] += __shfl_xor_sync(0xffffffffu, acc[d], 16);
  }
  lsum += __shfl_xor_sync(0xffffffffu, lsum, 8);
  lsum += __shfl_xor_sync(0xffffffffu, lsum, 16);
  if (sub == 0) {
#pragma unroll
    for (int d = 0; d < 8; ++d) s_acc[warp][8 * part + d] = acc[d];
  }
  if (lane == 0) { s_m[warp] = m_ref; s_l[warp] = lsum; }
  __syncthreads();
  float m = s_m[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, s_m[w]);
  float* out = p.ws + ((int64_t)split * p.B * p.H + bh) * 66;
  if (tid < 64) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) a = fmaf(s_acc[w][tid], (s_m[w] == -INFINITY) ? (s_l[w] != s_l[w] ? s_l[w] : 0.f) : exp2f(s_m[w] - m), a);
    out[2 + tid] = a;
  }
  if (tid == 0) {
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) l = fmaf(s_l[w], (s_m[w] == -INFINITY) ? (s_l[w] != s_l[w] ? s_l[w] : 0.f) : exp2f(s_m[w] - m), l);
    out[0] = m;
    out[1] = l;
  }
}

// One block per (batch, head): merge the splits in order, write y and lse, then add the weights.
template <bool kHalf>
__global__ void __launch_bounds__(NT) paged_join_kernel(PagedAttnParams p) {
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, tid = threadIdx.x;
  const int64_t N = keys_of(p, b), stride = (int64_t)p.B * p.H * 66;
  const float* rec = p.ws + (int64_t)bh * 66;
  float m = -INFINITY, l = 0.f, a = 0.f;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, rec[s * stride]);
  for (int s = 0; s < p.splits; ++s) {
    const float ms = rec[s * stride], ls = rec[s * stride + 1];
    const float sc = (ms == -INFINITY) ? (ls != ls ? ls : 0.f) : exp2f(ms - m);
    l = fmaf(ls, sc, l);
    if (tid < 64) a = fmaf(rec[s * stride + 2 + tid], sc, a);
  }
  const float lse = (N == 0) ? -INFINITY : m + log2f(l);
  if (tid < 64) {
    const float y = (N == 0) ? 0.f : a / l;
    const uint32_t w = pack2<kHalf>(y, 0.f);
    reinterpret_cast<uint16_t*>(p.y + 2 * ((int64_t)b * p.y_sb + (int64_t)h * p.y_sh))[tid] = (uint16_t)w;
  }
  if (tid == 0) {
    if (p.lse) p.lse[bh] = lse;
    if (N > 0 && !isfinite(lse) && p.status) atomicOr(p.status, SISA_ST_NONFINITE);
  }
  if (!p.weight_out) return;
  const float* xs = p.ws + (int64_t)p.splits * stride + (int64_t)bh * p.max_keys;
  for (int64_t j = tid; j < N; j += NT) {
    const int page = page_of(p.pg, b, j, nullptr);
    if (page < 0) continue;
    const int64_t at = page * p.pg.s_sp + h * p.pg.s_sh + (j & ((1 << p.pg.page_shift) - 1));
    p.weight_out[at] = p.pg.weight[at] + exp2f(xs[j] - lse);
  }
}

}  // namespace pat

int paged_attn_splits(int64_t B, int64_t H, int64_t max_keys) {
  int64_t s = (148 * 8 * 4 + B * H - 1) / (B * H);
  const int64_t most = (max_keys + pat::NT - 1) / pat::NT;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

cudaError_t launch_paged_attn(const PagedAttnParams& p, int dtype, cudaStream_t st) {
  dim3 grid(p.splits, p.B * p.H);
  if (dtype == 1) {
    pat::paged_split_kernel<true><<<grid, pat::NT, 0, st>>>(p);
    pat::paged_join_kernel<true><<<p.B * p.H, pat::NT, 0, st>>>(p);
  } else {
    pat::paged_split_kernel<false><<<grid, pat::NT, 0, st>>>(p);
    pat::paged_join_kernel<false><<<p.B * p.H, pat::NT, 0, st>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace sisa
