// paged_cache.cu - what a paged, bounded cache does around the attention that reads it: the slot whose
// key a new token replaces, the new token's write, and the cut of a prompt into pages.
#include <cuda_runtime.h>
#include <cstdint>

#include "sm100.cuh"
#include "gate_math.cuh"
#include "paged.h"

namespace sisa {
namespace pca {

constexpr int NT = 256, NW = NT / 32;

// ------------------------------------------------------------------------------------ evict
// One block per (batch, head): slots[b, h] = the slot j < budget of the least weight among the keys whose
// token is older than the `recent` newest (token < position - recent), the lowest slot where several
// weigh the same; -1 while the sequence holds fewer than budget keys. (weight, slot) is one 64-bit key,
// so the minimum does not depend on the order in which it is taken.
__global__ void __launch_bounds__(NT) paged_evict_kernel(PagedEvictParams p) {
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, tid = threadIdx.x;
  const int64_t pos = p.position[b];
  if (pos < p.budget) {
    if (tid == 0) p.slots[bh] = -1;
    return;
  }
  const int64_t newest = pos - p.recent;
  unsigned long long best = ~0ull;
  for (int64_t j = tid; j < p.budget; j += NT) {
    const int page = page_of(p.pg, b, j, p.status);
    if (page < 0) continue;
    const int64_t at = page * p.pg.s_sp + h * p.pg.s_sh + (j & ((1 << p.pg.page_shift) - 1));
    if (p.pg.token[at] >= newest) continue;
    const unsigned long long key = ((unsigned long long)weight_order(p.pg.weight[at]) << 32) | (unsigned)j;
    best = key < best ? key : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    best = other < best ? other : best;
  }
  __shared__ unsigned long long s_best[NW];
  if ((tid & 31) == 0) s_best[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < NW; ++w) best = s_best[w] < best ? s_best[w] : best;
    p.slots[bh] = best == ~0ull ? -1 : (int)(unsigned)best;
    if (best == ~0ull && p.status) atomicOr(p.status, SISA_ST_BAD_POS);
  }
}

// ------------------------------------------------------------------------------------ append
// One warp per (batch, head): the new token's recurrences g' = g - softplus(alpha), F' = F + logsigmoid(z),
// Phi' = Phi + theta, the rotation of c and b by Phi' (fp32, torch's separate products, one rounding), and
// the write of its key into one slot of the sequence's pages. An idle row (position < 0) keeps its state,
// writes no key and leaves zeros on the query side.
template <bool kHalf>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedAppendParams p) {
  const int w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (w >= p.B * p.H) return;
  const int b = w / p.H, h = w - b * p.H;
  const int64_t pos = p.position[b];
  const float* ci = p.carry_in + (int64_t)w * 18;
  float* co = p.carry_out + (int64_t)w * 18;
  int64_t slot = pos;
  if (p.slots) { const int s = p.slots[w]; if (s >= 0) slot = s; }
  int page = -1;
  if (pos >= 0) {
    if (slot < p.cap) page = page_of(p.pg, b, slot, lane == 0 ? p.status : nullptr);
    else if (lane == 0 && p.status) atomicOr(p.status, SISA_ST_BAD_POS);
  }
  const bool live = page >= 0;
  if (p.lengths && h == 0 && lane == 0) {
    const int64_t n = pos < 0 ? 0 : pos + 1;
    p.lengths[b] = (int)(p.budget > 0 && n > p.budget ? p.budget : n);
  }
  if (!live) {
    const float keep = lane < 18 ? ci[lane] : 0.f;
    if (lane < 18) co[lane] = keep;
    if (lane < 16) reinterpret_cast<uint32_t*>(p.c_out + (int64_t)w * 32)[lane] = 0u;
    if (lane == 16) p.g_out[w] = 0.f;
    if (lane == 17 && p.f_out) p.f_out[w] = 0.f;
    return;
  }
  const uint16_t* row = p.proj + (int64_t)b * p.proj_sb;
  auto to_f = [](uint16_t x) {
    if constexpr (kHalf) return __half2float(__ushort_as_half(x));
    else return __uint_as_float((uint32_t)x << 16);
  };
  auto to_lp = [](float x) -> uint16_t {
    if constexpr (kHalf) return __half_as_ushort(__float2half_rn(x));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  };
  const int64_t in = slot & ((1 << p.pg.page_shift) - 1);
  const int64_t at = page * p.pg.s_sp + h * p.pg.s_sh + in;
  reinterpret_cast<uint32_t*>(p.pg.k + 2 * (page * p.pg.k_sp + h * p.pg.k_sh + in * 64))[lane] =
      reinterpret_cast<const uint32_t*>(row + p.col_k + h * 64)[lane];
  reinterpret_cast<uint32_t*>(p.pg.v + 2 * (page * p.pg.v_sp + h * p.pg.v_sh + in * 64))[lane] =
      reinterpret_cast<const uint32_t*>(row + p.col_v + h * 64)[lane];
  if (lane < 16) {
    const float phin = to_f(row[p.col_th + h * 16 + lane]) + ci[lane];
    co[lane] = phin;
    const float cs = cosf(phin), sn = sinf(phin);
    const int e = 2 * lane;
    const float ce = to_f(row[p.col_c + h * 32 + e]), cd = to_f(row[p.col_c + h * 32 + e + 1]);
    const float be = to_f(row[p.col_b + h * 32 + e]), bd = to_f(row[p.col_b + h * 32 + e + 1]);
    reinterpret_cast<uint32_t*>(p.c_out + (int64_t)w * 32)[lane] =
        (uint32_t)to_lp(__fsub_rn(__fmul_rn(ce, cs), __fmul_rn(cd, sn))) |
        ((uint32_t)to_lp(__fadd_rn(__fmul_rn(ce, sn), __fmul_rn(cd, cs))) << 16);
    reinterpret_cast<uint32_t*>(p.pg.b + 2 * (page * p.pg.b_sp + h * p.pg.b_sh + in * 32))[lane] =
        (uint32_t)to_lp(__fsub_rn(__fmul_rn(be, cs), __fmul_rn(bd, sn))) |
        ((uint32_t)to_lp(__fadd_rn(__fmul_rn(be, sn), __fmul_rn(bd, cs))) << 16);
  } else if (lane == 16) {
    const float g = neg_softplus(to_f(row[p.col_a + h])) + ci[16];
    co[16] = g;
    p.g_out[w] = g;
    p.pg.g[at] = g;
  } else if (lane == 17) {
    const float f = p.z ? logsigmoid(p.z[(int64_t)b * p.z_sb + h]) + ci[17] : ci[17];
    co[17] = f;
    if (p.f_out) p.f_out[w] = f;
    if (p.pg.f) p.pg.f[at] = p.z ? f : 0.f;
  } else if (lane == 18) {
    if (p.pg.weight) p.pg.weight[at] = 0.f;
  } else if (lane == 19) {
    if (p.pg.token) p.pg.token[at] = (int)pos;
  }
}

// ------------------------------------------------------------------------------------ fill
// The kept keys of one (batch, head), ascending: the last `recent`, and of the rest the keep - recent of
// the largest weight, the earlier position where two weigh the same. A radix select over the ordered
// weights (eight bits a pass) finds the smallest kept weight T and how many of the keys at T are kept;
// a block scan then writes the kept positions in order.
__device__ __forceinline__ int block_scan_excl(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int c = s_warp[w];
    if (w < warp) base += c;
    total += c;
  }
  __syncthreads();
  return base + x - v;
}

__global__ void __launch_bounds__(NT) paged_select_kernel(PagedFillParams p) {
  const int bh = blockIdx.x, tid = threadIdx.x;
  int32_t* out = p.index + (int64_t)bh * p.keep;
  const float* wt = p.weight ? p.weight + (int64_t)bh * p.L : nullptr;
  const int64_t old = p.L - p.recent;              // positions [0, old) compete for keep - recent places
  __shared__ int s_hist[256], s_warp[NW];
  __shared__ uint32_t s_prefix;
  __shared__ int64_t s_left;
  uint32_t prefix = 0;
  int64_t left = p.keep - p.recent;                // places left among the keys that match the prefix
  if (wt && p.keep < p.L) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      s_hist[tid] = 0;
      __syncthreads();
      for (int64_t j = tid; j < old; j += NT) {
        const uint32_t u = weight_order(wt[j]);
        if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int64_t n = left;
        int d = 255;
        while (d > 0 && n > s_hist[d]) n -= s_hist[d--];
        s_prefix = prefix | ((uint32_t)d << shift);
        s_left = n;
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
      __syncthreads();
    }
  }
  const bool all = !wt || p.keep == p.L;
  int64_t done = 0, ties = 0;                       // kept so far, keys at the threshold so far
  for (int64_t j0 = 0; j0 < p.L; j0 += NT) {
    const int64_t j = j0 + tid;
    const uint32_t u = (!all && j < old) ? weight_order(wt[j]) : 0u;
    const bool tie = !all && j < old && u == prefix;
    int tot = 0, rank = 0;
    if (!all) {
      rank = block_scan_excl(tie ? 1 : 0, s_warp, tot);
    }
    const bool keep = j < p.L && (all || j >= old || u > prefix || (tie && ties + rank < left));
    int kept;
    const int at = block_scan_excl(keep ? 1 : 0, s_warp, kept);
    if (keep && done + at < p.keep) out[done + at] = (int)j;
    done += kept;
    ties += tot;
  }
}

// Eight lanes per kept key copy its rows (16 bytes a lane) and its plane values into slot r of the
// sequence's pages.
__global__ void __launch_bounds__(256) paged_gather_kernel(PagedFillParams p) {
  const int bh = blockIdx.y, b = bh / p.H, h = bh % p.H;
  const int64_t r = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const int part = threadIdx.x & 7;
  if (r >= p.keep) return;
  const int64_t j = p.index[(int64_t)bh * p.keep + r];
  const int page = page_of(p.pg, b, r, p.status);
  if (page < 0) return;
  const int64_t in = r & ((1 << p.pg.page_shift) - 1);
  reinterpret_cast<uint4*>(p.pg.k + 2 * (page * p.pg.k_sp + h * p.pg.k_sh + in * 64))[part] =
      reinterpret_cast<const uint4*>(p.k + 2 * (b * p.k_sb + h * p.k_sh + j * p.k_sl))[part];
  reinterpret_cast<uint4*>(p.pg.v + 2 * (page * p.pg.v_sp + h * p.pg.v_sh + in * 64))[part] =
      reinterpret_cast<const uint4*>(p.v + 2 * (b * p.v_sb + h * p.v_sh + j * p.v_sl))[part];
  if (part < 4)
    reinterpret_cast<uint4*>(p.pg.b + 2 * (page * p.pg.b_sp + h * p.pg.b_sh + in * 32))[part] =
        reinterpret_cast<const uint4*>(p.b + 2 * (b * p.b_sb + h * p.b_sh + j * p.b_sl))[part];
  const int64_t at = page * p.pg.s_sp + h * p.pg.s_sh + in;
  if (part == 4) p.pg.g[at] = p.g[b * p.g_sb + h * p.g_sh + j];
  if (part == 5 && p.pg.f) p.pg.f[at] = p.f ? p.f[b * p.f_sb + h * p.f_sh + j] : 0.f;
  if (part == 6 && p.pg.weight) p.pg.weight[at] = p.weight ? p.weight[(int64_t)bh * p.L + j] : 0.f;
  if (part == 7 && p.pg.token) p.pg.token[at] = (int)j;
}

}  // namespace pca

cudaError_t launch_paged_evict(const PagedEvictParams& p, cudaStream_t st) {
  pca::paged_evict_kernel<<<p.B * p.H, pca::NT, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_append(const PagedAppendParams& p, int dtype, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.B * p.H + 7) / 8);
  if (dtype == 1) pca::paged_append_kernel<true><<<grid, 256, 0, st>>>(p);
  else pca::paged_append_kernel<false><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_fill(const PagedFillParams& p, cudaStream_t st) {
  pca::paged_select_kernel<<<p.B * p.H, pca::NT, 0, st>>>(p);
  dim3 grid((unsigned)((p.keep + 31) / 32), p.B * p.H);
  pca::paged_gather_kernel<<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace sisa
