// key_weights.cu - the attention each prompt key received, on Blackwell tensor cores:
//   w_j = sum over queries i in [max(j, first), L) of 2^(x_ij - lse_i),
//   x_ij = log2e (q_i.k_j / 8 + lam_h exp(min(g_i - g_j, 0)) (c_i.b~_j) + (F_i - F_j)),
// with lse from the attention forward, so no running maximum is needed and every share is <= 1.
//
// CTA = 128 keys of one (batch, head), resident; it walks the 64-query tiles from its own diagonal (or from
// first) to the end. Warp roles:
//   warps 0-7  compute: a thread owns one key row (TMEM lane) and 32 of a tile's 64 query columns, so the
//              sum over queries is thread-local and the two halves meet once at the end,
//   warp 8     TMA producer of the Q, C and position tiles; its lanes also form the queries' additive terms,
//   warp 9     UMMA issuer and TMEM owner.
// Per tile S^T = K Q^T (M128 N64 K64) and U^T = B~ C^T (K32) land in tensor memory; the threads read them 16
// columns at a time, so that 64 registers do and three CTAs share an SM, whose GEMMs, loads and arithmetic
// overlap (two CTAs with two TMEM buffers each: the same time with all queries, 82 -> 96 us for the last 256
// queries of 8 x 16 heads x 4096, where a CTA lives for few tiles).
// Off the diagonal the decay is the product of three factors <= 1: the query's within its 64-row block (a
// stored plane), the one between the blocks (one per tile) and the key's to the end of its tile (one per
// thread). Per pair of elements that leaves five packed-fp32 instructions and two exponentials.
// Sums: a tile's 32 shares are added in two packed chains and then join the running sum, so a sum over
// 16384 queries is a chain of 256 additions and not of 16384.
// Bound: the exponential unit (16 a clock and SM) would need 119 us for the 5.4e8 pairs of 4 x 16 heads x
// 4096; 260 us measured, with the issue slots about 60 % and the exponential unit about half busy.
#include <cuda_runtime.h>
#include <type_traits>

#include "attn_common.cuh"
#include "key_weights.h"

namespace sisa {
namespace kwt {

constexpr int BK = 128, BQ = 64, NSTAGE = 3, NCW = 8;            // keys, queries per tile, stages, compute warps
constexpr int NG = NCW / 4, NC = BQ / NG;                        // warps per key row, query columns of each
constexpr int CH = 16;                                           // columns read at a time
constexpr uint32_t SZ_K = BK * 128, SZ_B = BK * 64;
constexpr uint32_t SZ_Q = BQ * 128, SZ_C = BQ * 64, SZ_POS = BQ * 16, SZ_LSE = BQ * 4;
constexpr uint32_t OFFS_C = SZ_Q, OFFS_POS = OFFS_C + SZ_C, OFFS_LSE = OFFS_POS + SZ_POS;
constexpr uint32_t SZ_STAGE = 14 * 1024;
static_assert(OFFS_LSE + SZ_LSE <= SZ_STAGE, "stage");
constexpr uint32_t OFF_K = 0, OFF_B = OFF_K + SZ_K, OFF_ST = OFF_B + SZ_B;
constexpr uint32_t OFF_SUM = OFF_ST + NSTAGE * SZ_STAGE, OFF_BAR = OFF_SUM + (NG - 1) * BK * 4;
constexpr uint32_t SMEM_BYTES = OFF_BAR + 256 + 1024;
static_assert(OFF_ST % 1024 == 0 && SZ_STAGE % 1024 == 0, "swizzle alignment");
static_assert(3 * (SMEM_BYTES + 1024) <= 228 * 1024, "three CTAs per SM");
constexpr uint32_t TMEM_COLS = 128;                              // S^T (64) and U^T (64)
constexpr int B_K = 0, B_QF = 1, B_QE = B_QF + NSTAGE, B_SF = B_QE + NSTAGE, B_SE = B_SF + 1;
static_assert((B_SE + 1) * 8 <= 128, "barriers end below the TMEM slot");
constexpr int NT = (NCW + 2) * 32;

template <bool kHalf>
__global__ void __launch_bounds__(NT, 3) key_weights_kernel(const __grid_constant__ KeyWeightParams p) {
  extern __shared__ uint8_t smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int bh, kt;
  tile_order(p.ntk, p.B * p.H, bh, kt);            // the first key tiles have the most queries
  const int b = bh / p.H, h = bh % p.H;
  const int L = p.L, k0 = kt * BK;
  const int i_begin = max(p.first, k0) / BQ * BQ;
  const int ntiles = (L - i_begin + BQ - 1) / BQ;  // >= 1: k0 < L and first < L

  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (sbase - raw);
  const uint32_t sK = sbase + OFF_K, sB = sbase + OFF_B;
  const uint32_t bar0 = sbase + OFF_BAR;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + OFF_BAR + 128);
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
  auto stage_addr = [&](int s) { return sbase + OFF_ST + (uint32_t)s * SZ_STAGE; };

  if (tid == 0) {
    mbar_init(BAR(B_K), 1);
    for (int s = 0; s < NSTAGE; ++s) {
      mbar_init(BAR(B_QF + s), 33);                // the TMA bytes and 32 lanes' query terms
      mbar_init(BAR(B_QE + s), NCW + 1);           // the compute warps and the UMMAs
    }
    mbar_init(BAR(B_SF), 1);
    mbar_init(BAR(B_SE), NCW);
    fence_barrier_init();
  }
  if (warp == NCW + 1) { tmem_alloc(smem_u32(tmem_slot), TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;

  if (warp == NCW) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      mbar_expect_tx(BAR(B_K), SZ_K + SZ_B);
      tma_load_4d(sK, &p.tm_k, BAR(B_K), 0, k0, h, b);
      tma_load_4d(sB, &p.tm_b, BAR(B_K), 0, k0, h, b);
    }
    // per query of the tile a_i = (F_i - F of the tile's first query) log2e - lse_i: taken relative to the
    // tile, the difference keeps the precision that F itself, a sum over the whole prompt, would cost
    const float* lse = p.lse + (int64_t)bh * L;
    const float* fpl = p.pos + (int64_t)bh * 4 * p.Lp + p.Lp;
    auto f_at = [&](int i) { return i < L ? __ldg(fpl + i) : 0.f; };
    auto lse_at = [&](int i) { return i < L ? __ldg(lse + i) : 0.f; };
    float f0 = f_at(i_begin + lane), f1 = f_at(i_begin + lane + 32);
    float n0 = lse_at(i_begin + lane), n1 = lse_at(i_begin + lane + 32);
    int n = 0;
    for (; n < ntiles; ++n) {
      const int s = n % NSTAGE, i0 = i_begin + n * BQ;
      if (n >= NSTAGE && !warp_wait<true>(BAR(B_QE + s), ((n / NSTAGE) - 1) & 1, p.status)) break;
      const uint32_t st = stage_addr(s);
      if (lane == 0) {
        mbar_expect_tx(BAR(B_QF + s), SZ_Q + SZ_C + SZ_POS);
        tma_load_4d(st, &p.tm_q, BAR(B_QF + s), 0, i0, h, b);
        tma_load_4d(st + OFFS_C, &p.tm_c, BAR(B_QF + s), 0, i0, h, b);
        tma_load_3d(st + OFFS_POS, &p.tm_pos, BAR(B_QF + s), i0, 0, bh);
      }
      float* nl = reinterpret_cast<float*>(gbase + OFF_ST + s * SZ_STAGE + OFFS_LSE);
      const float fr = __shfl_sync(0xffffffffu, f0, 0);
      nl[lane] = fmaf(f0 - fr, kLOG2E, -n0);
      nl[lane + 32] = fmaf(f1 - fr, kLOG2E, -n1);
      mbar_arrive(BAR(B_QF + s));
      f0 = f_at(i0 + BQ + lane);
      f1 = f_at(i0 + BQ + lane + 32);
      n0 = lse_at(i0 + BQ + lane);                 // the next tile's, in flight while this warp waits
      n1 = lse_at(i0 + BQ + lane + 32);
    }
    if (n < ntiles) {                              // a wait ran out: let the copies in flight land before leaving
      warp_wait<true>(BAR(B_K), 0, p.status);
      for (int m = n - NSTAGE; m < n; ++m) warp_wait<true>(BAR(B_QF + m % NSTAGE), (m / NSTAGE) & 1, p.status);
    }
  } else if (warp == NCW + 1) {
    // ------------------------------------------------------------------ UMMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc(128, 64, kHalf ? 0 : 1, 0, 0);
      const bool ok = mbar_wait<true>(BAR(B_K), 0, p.status);
      int n = 0;
      for (; ok && n < ntiles; ++n) {
        const int s = n % NSTAGE;
        if (!mbar_wait<true>(BAR(B_QF + s), (n / NSTAGE) & 1, p.status)) break;
        if (n >= 1 && !mbar_wait<true>(BAR(B_SE), (n - 1) & 1, p.status)) break;
        tc_fence_after();
        const uint32_t st = stage_addr(s), tS = tbase, tU = tbase + 64;
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_ss(tS, desc_k128(sK + k * 32), desc_k128(st + k * 32), idesc, k > 0);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          umma_ss(tU, desc_k64(sB + k * 32), desc_k64(st + OFFS_C + k * 32), idesc, k > 0);
        umma_commit(BAR(B_SF));
        umma_commit(BAR(B_QE + s));
      }
      // (the same for the UMMAs, whose tensor memory is freed below)
      if (n < ntiles && n > 0) mbar_wait<true>(BAR(B_SF), (n - 1) & 1, p.status);
    }
  } else {
    // ------------------------------------------------------------------ compute
    const int r = tid & 127, grp = warp >> 2;      // key row of the tile, which NC query columns
    const int j = k0 + r;
    const float* posbh = p.pos + (int64_t)bh * 4 * p.Lp;
    const int jj = min(j, L - 1), je = min(k0 + BK, L) - 1;
    const float gj = posbh[jj], fj = posbh[p.Lp + jj], gend = posbh[je];
    const float lam2 = p.lam[h] * kLOG2E;
    const float cj = lam2 * exp2f(fmin_nan((gend - gj) * kLOG2E, 0.f));
    const float2 c1 = bcast2(kScale * kLOG2E);
    float2 total = bcast2(0.f);
    bool ok = true;
    for (int n = 0; n < ntiles; ++n) {
      const int s = n % NSTAGE, i0 = i_begin + n * BQ;
      // the scores, and the query terms that the producer's lanes stored
      if (!warp_wait_tested<true>(BAR(B_SF), n & 1, p.status) ||
          !warp_wait_tested<true>(BAR(B_QF + s), (n / NSTAGE) & 1, p.status)) { ok = false; break; }
      tc_fence_after();
      const float* q = reinterpret_cast<const float*>(gbase + OFF_ST + s * SZ_STAGE + OFFS_POS);
      const float4* qr4 = reinterpret_cast<const float4*>(q + 2 * BQ) + grp * (NC / 4);       // decay within the block
      const float4* ql4 = reinterpret_cast<const float4*>(q + 4 * BQ) + grp * (NC / 4);       // a_i
      const bool off = i0 >= k0 + BK;              // off the diagonal
      const float2 cf = bcast2((q[BQ] - fj) * kLOG2E);
      float2 t0 = bcast2(0.f), t1 = bcast2(0.f);
#pragma unroll
      for (int ch = 0; ch < NC; ch += CH) {
        float sv[CH], uv[CH];
        tmem_ld16(tmem_addr(tbase, warp & 3, grp * NC + ch), sv);
        tmem_ld16(tmem_addr(tbase, warp & 3, 64 + grp * NC + ch), uv);
        tmem_wait_ld();
        if (ch + CH == NC) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(B_SE));
        }
        const int c0 = i0 + grp * NC + ch;         // this thread's first query
        // the decay by factors. kMask: the tile reaches before `first` or past L
        auto factored = [&](auto mask) {
          constexpr bool kMask = decltype(mask)::value;
          const float2 cm = bcast2(cj * exp2f(fmin_nan((q[0] - gend) * kLOG2E, 0.f)));
  #pragma unroll
          for (int c = 0; c < CH / 4; ++c) {
            const float4 r4 = qr4[c + ch / 4], l4 = ql4[c + ch / 4];
  #pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 rf = e ? make_float2(r4.z, r4.w) : make_float2(r4.x, r4.y);
              const float2 a = e ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y);
              const int at = 4 * c + 2 * e;
              const float2 d = fma2(mul2(make_float2(uv[at], uv[at + 1]), rf), cm, add2(a, cf));
              const float2 x = fma2(make_float2(sv[at], sv[at + 1]), c1, d);
              float2 pe = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              if constexpr (kMask) {
                if (c0 + at < p.first || c0 + at >= L) pe.x = 0.f;
                if (c0 + at + 1 < p.first || c0 + at + 1 >= L) pe.y = 0.f;
              }
              if (e) t1 = add2(t1, pe); else t0 = add2(t0, pe);
            }
          }
        };
        if (off) {
          if (i0 >= p.first && i0 + BQ <= L) factored(std::false_type{});
          else factored(std::true_type{});
        } else if (c0 + CH > k0 + (warp & 3) * 32) {
          // on the diagonal: pairwise decay, shares of later queries only (a warp whose keys all come after its
          // queries has none)
          const float* qg = q + grp * NC + ch;
  #pragma unroll
          for (int c = 0; c < CH; ++c) {
            const int i = c0 + c;
            const float dec = ex2_approx(fmin_nan((qg[c] - gj) * kLOG2E, 0.f));
            const float x = fmaf(sv[c], kScale * kLOG2E, fmaf(uv[c] * dec, lam2, cf.x + qg[4 * BQ + c]));
            const float pe = (i >= j && i >= p.first && i < L) ? ex2_approx(x) : 0.f;
            if (c & 1) t0.y += pe; else t0.x += pe;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(B_QE + s));
      total = add2(total, add2(t0, t1));
    }
    float* sums = reinterpret_cast<float*>(gbase + OFF_SUM);
    const float mine = total.x + total.y;
    if (grp) sums[(grp - 1) * BK + r] = mine;
    named_bar_sync(1, NCW * 32);
    if (!grp && j < L) {
      float w = mine;
#pragma unroll
      for (int e = 0; e < NG - 1; ++e) w += sums[e * BK + r];
      p.w[(int64_t)bh * L + j] = w;
      if (ok && !isfinite(w) && p.status) atomicOr(p.status, SISA_ST_NONFINITE);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == NCW + 1) {
    tc_fence_after();
    tmem_dealloc(tbase, TMEM_COLS);
  }
#undef BAR
}

}  // namespace kwt

cudaError_t launch_key_weights(const KeyWeightParams& p, int dtype, cudaStream_t st) {
  using namespace kwt;
  auto* kernel = dtype == 1 ? key_weights_kernel<true> : key_weights_kernel<false>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
  if (e != cudaSuccess) return e;
  kernel<<<dim3(p.ntk, p.B * p.H), NT, SMEM_BYTES, st>>>(p);
  return cudaGetLastError();
}

}  // namespace sisa
