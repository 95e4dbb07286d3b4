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

__device__ __forceinline__ int cluster_blocks() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return (int)n;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
// The 64-bit word of block `rank` of this cluster at the shared-memory place of `p`.
__device__ __forceinline__ unsigned long long cluster_load(const unsigned long long* p, int rank) {
  uint32_t addr;
  unsigned long long v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// ------------------------------------------------------------------------------------ evict
// slots[b, h] = the slot j < budget of the least weight among the keys whose token is older than the `recent`
// newest (token < position - recent), the lowest slot where several weigh the same; -1 while the sequence
// holds fewer than budget keys. (weight, slot) is one 64-bit number, so the minimum does not depend on the
// order in which it is taken.
// Bound by memory: 8 bytes per key. A thread takes four slots at a time (16-byte loads of both planes), two such
// steps in flight; a cluster of blocks shares a unit when there are few units, and its first block takes
// the minimum over the others' through distributed shared memory. 64 x 16 units of 8192 slots (67 MB): 13.4 us where
// the planes are still in L2, 18.1 us = 3.7 TB/s where five other layers' planes have passed in between. In L2, one
// step in flight 14.5 us; with 64-bit comparisons per slot 16.6 us (four steps: 20.6 us); the first version, one
// slot per thread and step, 38 us.
constexpr int EVICT_CLUSTER = 8;                 // portable cluster size
__global__ void __launch_bounds__(NT) paged_evict_kernel(PagedEvictParams p) {
  const int cs = cluster_blocks(), rank = blockIdx.x % cs;
  const int bh = blockIdx.x / cs, b = bh / p.H, h = bh % p.H, tid = threadIdx.x;
  const int64_t pos = p.position[b];
  __shared__ unsigned long long s_best[NW + 1];
  unsigned long long best = ~0ull;
  if (pos >= p.budget) {                         // uniform over the cluster
    const int64_t newest = pos - p.recent;
    const int64_t step = (int64_t)cs * NT * 4;
    struct Four { float4 w; int4 t; bool ok; };
    auto load = [&](int64_t j) {
      Four f;
      f.ok = false;
      if (j >= p.budget) return f;
      const int page = page_of(p.pg, b, j, p.status);
      if (page < 0) return f;
      const int64_t at = page * p.pg.s_sp + h * p.pg.s_sh + (j & ((1 << p.pg.page_shift) - 1));
      f.w = __ldg(reinterpret_cast<const float4*>(p.pg.weight + at));
      f.t = __ldg(reinterpret_cast<const int4*>(p.pg.token + at));
      f.ok = true;
      return f;
    };
    // a thread meets its slots in ascending order, so the first of the least weight is kept by a strict
    // comparison; 0xffffffff is above the order of every weight
    uint32_t least = 0xffffffffu, slot = 0;
    auto take = [&](const Four& f, int64_t j) {
      if (!f.ok) return;
      const float w[4] = {f.w.x, f.w.y, f.w.z, f.w.w};
      const int t[4] = {f.t.x, f.t.y, f.t.z, f.t.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u = weight_order(w[e]);
        if (u < least && t[e] < newest && j + e < p.budget) { least = u; slot = (uint32_t)j + e; }
      }
    };
    for (int64_t j = ((int64_t)rank * NT + tid) * 4; j < p.budget; j += 2 * step) {
      const Four f0 = load(j), f1 = load(j + step);
      take(f0, j);
      take(f1, j + step);
    }
    if (least != 0xffffffffu) best = ((unsigned long long)least << 32) | slot;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other < best ? other : best;
    }
    if ((tid & 31) == 0) s_best[tid >> 5] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < NW; ++w) best = s_best[w] < best ? s_best[w] : best;
      s_best[NW] = best;
    }
  }
  if (cs > 1) cluster_sync();
  if (rank == 0 && tid == 0) {
    for (int r = 1; r < cs && pos >= p.budget; ++r) {
      const unsigned long long other = cluster_load(&s_best[NW], r);
      best = other < best ? other : best;
    }
    p.slots[bh] = best == ~0ull ? -1 : (int)(unsigned)best;
    if (pos >= p.budget && best == ~0ull && p.status) atomicOr(p.status, SISA_ST_BAD_POS);
  }
  if (cs > 1) cluster_sync();                    // the others' shared memory stays until it has been read
}

// ------------------------------------------------------------------------------------ append
// One warp per (batch, head): the new token's recurrences g' = g - softplus(alpha), F' = F + logsigmoid(z),
// Phi' = Phi + theta, the rotation of c and b by Phi' (fp32, torch's separate products, one rounding), and
// the write of its key into one slot of the sequence's pages. An idle row (position < 0) keeps its state,
// writes no key and leaves zeros on the query side. Bound by latency: about 1 KB per (sequence, head), 5.5-7 us
// for one sequence and for 64 x 16 heads, most of it the chain position -> page -> slot.
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
// the largest weight, the earlier position where two weigh the same. One block per unit:
//   1. a radix select over the ordered weights (11 + 11 + 10 bits) finds the smallest kept weight T and how
//      many of the keys at T are kept; it ends where a digit is kept whole, and after the first digit reads
//      only the keys that share it;
//   2. per 32-key group the kept keys above T and the ties are counted, two block scans (ties first: how
//      many of them a group keeps depends on those before it) place the groups, and the kept positions
//      are written in order.
// The weights of up to SEL_SMEM keys are ordered once into shared memory; longer prompts are read again
// from L2 in each pass. Bound by instructions (72 % of the issue slots): 20 us for 256 units of 8192 keys, 6 us for
// 16 units of 1000.
constexpr int ST = 1024, SW = ST / 32, SEL_SMEM = 40960;
static_assert(SW <= 32 && 2048 % ST == 0, "scan and bins");
constexpr int BINS = 2048;

// Exclusive scan over the block's threads; total in every thread.
__device__ __forceinline__ int scan_excl(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  const int c = lane < SW ? s_warp[lane] : 0;
  int y = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  total = __shfl_sync(0xffffffffu, y, 31);
  const int base = __shfl_sync(0xffffffffu, y - c, warp);
  __syncthreads();
  return base + x - v;
}

__global__ void __launch_bounds__(ST) paged_select_kernel(PagedFillParams p) {
  extern __shared__ uint32_t s_key[];            // ordered weights of positions [0, old) when they fit
  __shared__ int s_hist[BINS], s_warp[32];
  // the candidates of the later passes; then per 32-key group: keys surely kept, ties, first place, ties before
  __shared__ uint32_t s_buf[4 * ST];
  __shared__ uint32_t s_digit;
  __shared__ int s_left, s_in, s_count;
  asm volatile("griddepcontrol.launch_dependents;");
  const int bh = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t below = (1u << lane) - 1;
  int32_t* out = p.index + (int64_t)bh * p.keep;
  const int L = (int)p.L, old = (int)(p.L - p.recent);   // positions [0, old) compete for keep - recent places
  const float* wt = p.weight + (int64_t)bh * p.L;
  const bool in_smem = old <= SEL_SMEM;
  if (in_smem) {
    for (int j = tid; j < old; j += ST) s_key[j] = weight_order(__ldg(wt + j));
  }
  auto key_at = [&](int j) { return in_smem ? s_key[j] : weight_order(__ldg(wt + j)); };
  // with no place left nothing but the newest is kept: no key is above the largest order
  uint32_t prefix = p.keep == p.recent ? 0xffffffffu : 0u;
  int left = (int)(p.keep - p.recent);           // places left among the keys that match the prefix
  int cand = -1;                                 // candidates in s_buf, -1: every key is looked at
  if (tid == 0) s_count = 0;
  if (left > 0) {
    int shift = 32;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10, above = shift;
      shift -= bits;
      for (int i = tid; i < BINS; i += ST) s_hist[i] = 0;
      __syncthreads();
      const uint32_t digits = (1u << bits) - 1;
      if (cand >= 0) {
        for (int j = tid; j < cand; j += ST) {
          const uint32_t u = s_buf[j];
          if ((u >> above) == (prefix >> above)) atomicAdd(&s_hist[(u >> shift) & digits], 1);
        }
      } else {
        for (int j = tid; j < old; j += ST) {
          const uint32_t u = key_at(j);
          if (above == 32 || (u >> above) == (prefix >> above)) atomicAdd(&s_hist[(u >> shift) & digits], 1);
        }
      }
      __syncthreads();
      // thread t holds BINS / ST bins from BINS - 1 - t BINS / ST down: the scan runs from the largest digit
      const int d = BINS - 1 - (BINS / ST) * tid;
      int own = 0, total;
#pragma unroll
      for (int i = 0; i < BINS / ST; ++i) own += s_hist[d - i];
      int over = scan_excl(own, s_warp, total);
      if (over < left && left <= over + own) {   // the wanted digit is one of this thread's
        int i = 0;
        while (left > over + s_hist[d - i]) over += s_hist[d - i++];
        s_digit = d - i;
        s_left = left - over;
        s_in = s_hist[d - i];
      }
      __syncthreads();
      prefix |= s_digit << shift;
      left = s_left;
      const int in = s_in;                       // keys with this digit
      if (left == in && prefix > 0) {            // all of them are kept: no need to look further into the digit
        --prefix;
        left = 0;
        break;
      }
      if (pass == 0 && in <= 4 * ST) {           // few are left to tell apart: the later passes read only them
        for (int j0 = 0; j0 < old; j0 += ST) {
          const int j = j0 + tid;
          const uint32_t u = j < old ? key_at(j) : 0u;
          const bool is = j < old && (u >> shift) == (prefix >> shift);
          const uint32_t m = __ballot_sync(0xffffffffu, is);
          int at = 0;
          if (lane == 0 && m) at = atomicAdd(&s_count, __popc(m));
          at = __shfl_sync(0xffffffffu, at, 0);
          at += __popc(m & below);
          if (is && at < 4 * ST) s_buf[at] = u;
        }
        cand = in;
      }
      // (the next pass's first barrier keeps the shared words until every thread has read them)
    }
  }
  __syncthreads();
  uint32_t* s_sure = s_buf;
  uint32_t* s_tie = s_buf + ST;
  int* s_base = reinterpret_cast<int*>(s_buf + 2 * ST);
  int* s_before = reinterpret_cast<int*>(s_buf + 3 * ST);
  int done = 0, ties = 0;                        // kept, and keys at T, in the chunks before
  for (int j0 = 0; j0 < L; j0 += ST * 32) {
    // group g of the chunk holds 32 consecutive positions
    const int groups = min(ST, (L - j0 + 31) / 32);
    for (int g = warp; g < groups; g += SW) {
      const int j = j0 + g * 32 + lane;
      const uint32_t u = j < old ? key_at(j) : 0u;
      const uint32_t sure = __ballot_sync(0xffffffffu, j < L && (j >= old || u > prefix));
      const uint32_t tie = __ballot_sync(0xffffffffu, j < old && u == prefix);
      if (lane == 0) { s_sure[g] = sure; s_tie[g] = tie; }
    }
    __syncthreads();
    int tot_tie, tot;
    const int nt = tid < groups ? __popc(s_tie[tid]) : 0, ns = tid < groups ? __popc(s_sure[tid]) : 0;
    const int tb = ties + scan_excl(nt, s_warp, tot_tie);
    s_base[tid] = done + scan_excl(ns + max(0, min(nt, left - tb)), s_warp, tot);
    s_before[tid] = tb;
    __syncthreads();
    for (int g = warp; g < groups; g += SW) {
      const uint32_t sure = s_sure[g], tie = s_tie[g];
      const bool keep = ((sure >> lane) & 1) || (((tie >> lane) & 1) && s_before[g] + __popc(tie & below) < left);
      const uint32_t kept = tie ? __ballot_sync(0xffffffffu, keep) : sure;
      const int at = s_base[g] + __popc(kept & below);
      if (keep && at < (int)p.keep) out[at] = j0 + g * 32 + lane;
    }
    __syncthreads();
    done += tot;
    ties += tot_tie;
  }
}

// 32 kept keys of one unit per block: eight lanes per key copy its rows (16 bytes a lane), 32 threads its
// plane values, into the sequence's pages. The units are the fast grid dimension, so the blocks in flight
// read the same part of the prompt for all heads, whose rows lie side by side in the projection. (Two keys
// a lane: 101 instead of 97 us for 16 x 16 units of 8192 -> 2048 keys, four: 122 us.)
constexpr int GK = 32;
__global__ void __launch_bounds__(256, 8) paged_gather_kernel(PagedFillParams p) {
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, tid = threadIdx.x, part = tid & 7;
  const int32_t* index = p.index + (int64_t)bh * p.keep;
  bool waited = false;
  for (int64_t r0 = (int64_t)blockIdx.y * GK; r0 < p.keep; r0 += (int64_t)gridDim.y * GK) {
    const int64_t r = r0 + (tid >> 3);
    const int page = r < p.keep ? page_of(p.pg, b, r, p.status) : -1;
    if (!waited) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      waited = true;
    }
    const int j = page < 0 ? -1 : (p.index ? index[r] : (int)r);
    if ((unsigned)j < (unsigned)p.L) {           // (an index outside the prompt cannot arise; it would be left out)
      const int64_t in = r & ((1 << p.pg.page_shift) - 1);
      const uint4 k = __ldg(reinterpret_cast<const uint4*>(p.k + 2 * (b * p.k_sb + h * p.k_sh + j * p.k_sl)) + part);
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.v + 2 * (b * p.v_sb + h * p.v_sh + j * p.v_sl)) + part);
      uint4 m = make_uint4(0, 0, 0, 0);
      if (part < 4) m = __ldg(reinterpret_cast<const uint4*>(p.b + 2 * (b * p.b_sb + h * p.b_sh + j * p.b_sl)) + part);
      reinterpret_cast<uint4*>(p.pg.k + 2 * (page * p.pg.k_sp + h * p.pg.k_sh + in * 64))[part] = k;
      reinterpret_cast<uint4*>(p.pg.v + 2 * (page * p.pg.v_sp + h * p.pg.v_sh + in * 64))[part] = v;
      if (part < 4) reinterpret_cast<uint4*>(p.pg.b + 2 * (page * p.pg.b_sp + h * p.pg.b_sh + in * 32))[part] = m;
    }
    if (tid < GK && r0 + tid < p.keep) {
      const int64_t rr = r0 + tid;
      const int j = p.index ? index[rr] : (int)rr, pp = page_of(p.pg, b, rr, nullptr);
      if (pp >= 0 && (unsigned)j < (unsigned)p.L) {
        const int64_t at = pp * p.pg.s_sp + h * p.pg.s_sh + (rr & ((1 << p.pg.page_shift) - 1));
        const float g = __ldg(p.g + b * p.g_sb + h * p.g_sh + j);
        const float f = p.f ? __ldg(p.f + b * p.f_sb + h * p.f_sh + j) : 0.f;
        const float w = p.weight ? __ldg(p.weight + (int64_t)bh * p.L + j) : 0.f;
        p.pg.g[at] = g;
        if (p.pg.f) p.pg.f[at] = f;
        if (p.pg.weight) p.pg.weight[at] = w;
        if (p.pg.token) p.pg.token[at] = j;
      }
    }
  }
}

}  // namespace pca

cudaError_t launch_paged_evict(const PagedEvictParams& p, cudaStream_t st) {
  // blocks per unit: enough for four blocks per SM, each with at least one step of 1024 slots
  const int64_t units = (int64_t)p.B * p.H;
  int cs = 1;
  while (cs < pca::EVICT_CLUSTER && units * cs < 148 * 4 && (int64_t)cs * pca::NT * 4 < p.budget) cs *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * cs));
  cfg.blockDim = dim3(pca::NT);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pca::paged_evict_kernel, p);
}

cudaError_t launch_paged_append(const PagedAppendParams& p, int dtype, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.B * p.H + 7) / 8);
  if (dtype == 1) pca::paged_append_kernel<true><<<grid, 256, 0, st>>>(p);
  else pca::paged_append_kernel<false><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_fill(PagedFillParams p, cudaStream_t st) {
  const bool choose = p.keep < p.L;
  if (choose) {
    const int64_t old = p.L - p.recent;
    const size_t smem = old <= pca::SEL_SMEM ? (size_t)old * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute(pca::paged_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         pca::SEL_SMEM * 4);
    if (e != cudaSuccess) return e;
    pca::paged_select_kernel<<<p.B * p.H, pca::ST, smem, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  } else {
    p.index = nullptr;                           // every key is kept: slot r takes position r
  }
  const int64_t chunks = (p.keep + pca::GK - 1) / pca::GK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.B * p.H, (unsigned)(chunks < 65535 ? chunks : 65535));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its blocks wait for the choice themselves
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = choose ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, pca::paged_gather_kernel, p);
}

}  // namespace sisa
