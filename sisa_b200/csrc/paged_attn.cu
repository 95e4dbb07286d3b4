// paged_attn.cu - attention of one new token per sequence over its paged keys, split over the keys and joined.
//
// For every sequence b with n_b keys (slots 0 .. n_b - 1 of its pages, in any order) and head h:
//   x_j = log2e (q.k_j / 8 + lam_h exp(min(g_q - g_j, 0)) (c.b~_j) + (F_q - F_j)),
//   y = sum_j 2^(x_j - lse) v_j,  lse = log2 sum_j 2^x_j,  and optionally weight_j += 2^(x_j - lse).
// A row with no keys, or whose keys are all left out (table entries that name no page) or all score -inf,
// gives y = 0, lse = -inf and no shares.
//
// HBM-bound: 328 bytes per key and head (k, v, b~ in 16 bits, g and F in 32), 320 flops. Work is cut into
// tiles of 32 keys; the tiles of all (sequence, head) units lie in one line, and each of a fixed number of
// warps takes an equal run of it, so sequences of any mix of lengths load every SM alike. A warp is on its
// own: it fills a ring of stages in shared memory by bulk copies (one lane per operand, rows of a page are
// dense), reads each tile once, keeps the running maximum (moved only when a key exceeds it by 2^8), the
// sum and the 64 output sums in registers, and meets no block-wide barrier before its run is done. Eight lanes share a key
// (16 bytes of its rows each), so a tile is eight groups of four keys; the eight partial dot products of a
// lane are summed by a reduce-scatter over the eight lanes, after which every lane owns one key's score and
// the exponentials are taken once per key.
// A unit inside one warp's run is finished there. The pieces of the others are merged at the end of the CTA,
// whose warps' runs are neighbours; what reaches past the CTA leaves as (m, l, acc) records, at most two per
// CTA, that paged_join_kernel merges in order (deterministic, no atomics). With weights, the scores are kept
// in the workspace (4 bytes per key) and paged_weights_kernel adds the shares once lse is known.
//
// Measured (B200, a copy moves 6.55 TB/s): 64 sequences of 8192 keys x 16 heads 404 us = 6.81 TB/s, with weights
// 455-468 us = 6.1 TB/s; one of 131,071 keys x 16 heads 118-121 us = 5.7 TB/s, of which about 10 us are start-up and
// join.
// Ten warps per SM with two stages each: four warps with five stages (one CTA per SM) took 504 us on the first
// case before the waves, since a lone warp per scheduler hides none of its own latency.
#include <cuda_runtime.h>
#include <cstdint>

#include "attn_common.cuh"
#include "paged.h"

namespace sisa {
namespace pat {

constexpr int TK = 32;                          // keys per tile
constexpr int NW = 5, NSTAGE = 2;               // warps per CTA, ring stages per warp; two CTAs per SM
constexpr int NCTA = 148 * 16;                  // eight waves: SMs stream at different rates, and the ones
                                                // that are done take the next CTA
constexpr int UNIT_KEYS = 512;                  // tables up to this many keys: one CTA per unit (see launch)
constexpr int NWORK = NCTA * NW, WMIN = 296 * NW, GRAIN = 16;
constexpr uint32_t OFF_V = TK * 128, OFF_B = OFF_V + TK * 128, OFF_G = OFF_B + TK * 64, OFF_F = OFF_G + TK * 4;
constexpr int REC = 68;                         // floats of a record: m, l, 2 unused, acc[64]
constexpr uint32_t SZ_STAGE = OFF_F + TK * 4;   // 10,496 bytes
constexpr uint32_t SZ_WARP = NSTAGE * SZ_STAGE;
constexpr uint32_t OFF_REC = NW * SZ_WARP, OFF_BAR = OFF_REC + NW * 2 * REC * 4, OFF_MASK = OFF_BAR + NW * NSTAGE * 8;
constexpr uint32_t SMEM_BYTES = OFF_MASK + NW * NSTAGE * 4 + 128;
static_assert(SZ_STAGE % 128 == 0 && 2 * (SMEM_BYTES + UNIT_KEYS * 4 + 256 + 1024) <= 228 * 1024, "shared memory");

__device__ __forceinline__ int64_t keys_of(const PagedAttnParams& p, int b) {
  const int64_t n = __ldg(p.lengths + b);
  return n < 0 ? 0 : (n > p.max_keys ? p.max_keys : n);
}
__device__ __forceinline__ int64_t tiles_of(const PagedAttnParams& p, int b) { return (keys_of(p, b) + TK - 1) / TK; }

// Tiles per head of the sequences before b (all of them with b = B), computed by one warp.
__device__ __forceinline__ int64_t tiles_before(const PagedAttnParams& p, int b, int64_t& all) {
  int64_t before = 0, total = 0;
  for (int i = threadIdx.x & 31; i < p.B; i += 32) {
    const int64_t t = tiles_of(p, i);
    total += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  all = total;
  return before;
}

// The line is shared by one worker (warp) per tile while there are few tiles, then by the warps of one wave,
// and beyond GRAIN tiles a worker by more whole waves, up to eight; none has an empty run. Worker w takes the
// tiles [run_start(w), run_start(w + 1)); worker_of is its inverse.
__host__ __device__ __forceinline__ int64_t workers(int64_t tiles) {
  if (tiles < WMIN) return tiles;
  const int64_t waves = tiles / (WMIN * GRAIN);
  return waves < 1 ? WMIN : (waves < 8 ? waves * WMIN : NWORK);
}
__device__ __forceinline__ int64_t run_start(int64_t w, int64_t tiles) { return w * tiles / workers(tiles); }
__device__ __forceinline__ int worker_of(int64_t x, int64_t tiles) {
  return (int)(((x + 1) * workers(tiles) - 1) / tiles);
}

// A place in the line: tile t of the T tiles of (b, h).
struct Cursor {
  int b, h;
  int64_t t, T, n;
  __device__ __forceinline__ void load(const PagedAttnParams& p) { n = keys_of(p, b); T = (n + TK - 1) / TK; }
  // The next tile of the line (the caller knows that there is one).
  __device__ __forceinline__ void next(const PagedAttnParams& p) {
    if (++t < T) return;
    t = 0;
    if (++h < p.H) return;
    h = 0;
    do { ++b; load(p); } while (T == 0);
  }
};

// The cursor of tile x, found by one warp.
__device__ __forceinline__ Cursor find_tile(const PagedAttnParams& p, int64_t x) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  for (int b0 = 0;; b0 += 32) {
    const int64_t t = b0 + lane < p.B ? tiles_of(p, b0 + lane) : 0;
    int64_t incl = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int64_t lo = (base + incl - t) * p.H;
    const uint32_t hit = __ballot_sync(0xffffffffu, t > 0 && x >= lo && x < lo + t * p.H);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t T = __shfl_sync(0xffffffffu, t, src), rem = x - __shfl_sync(0xffffffffu, lo, src);
      Cursor c;
      c.b = b0 + src;
      c.h = (int)(rem / T);
      c.t = rem - c.h * T;
      c.load(p);
      return c;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
}

// A bulk copy whose lines L2 may drop first: the keys are read once, and what should stay in L2 is the
// scores that the weights pass reads back.
__device__ __forceinline__ uint64_t policy_evict_first() {
  uint64_t pol;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
  return pol;
}
__device__ __forceinline__ void bulk_load_hint(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
      ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(pol) : "memory");
}

template <bool kHalf>
__device__ __forceinline__ float2 unpack2(uint32_t w) { return make_float2(unpack_lo<kHalf>(w), unpack_hi<kHalf>(w)); }

// Eight values per lane summed over the eight lanes of a key group: lane `part` gets the sum of value part.
__device__ __forceinline__ float reduce_scatter8(const float (&v)[8], int part) {
  float a[4], c[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool hi = part & 4;
    a[i] = (hi ? v[i + 4] : v[i]) + __shfl_xor_sync(0xffffffffu, hi ? v[i] : v[i + 4], 4);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool hi = part & 2;
    c[i] = (hi ? a[i + 2] : a[i]) + __shfl_xor_sync(0xffffffffu, hi ? a[i] : a[i + 2], 2);
  }
  const bool hi = part & 1;
  return (hi ? c[1] : c[0]) + __shfl_xor_sync(0xffffffffu, hi ? c[0] : c[1], 1);
}

// A softmax sum held by a warp: maximum, sum, and head dims 2 lane, 2 lane + 1 of the weighted values.
struct Sum {
  float m, l;
  float2 a;
  __device__ __forceinline__ void clear() { m = -INFINITY; l = 0.f; a = make_float2(0.f, 0.f); }
  __device__ __forceinline__ void add(float2 ml, float2 v) {
    const float mn = fmaxf(m, ml.x), mb = mn == -INFINITY ? 0.f : mn;
    const float s0 = exp2f(m - mb), s1 = exp2f(ml.x - mb);
    l = fmaf(ml.y, s1, l * s0);
    a = fma2(v, bcast2(s1), mul2(a, bcast2(s0)));
    m = mn;
  }
  __device__ __forceinline__ void add(const float* rec) {
    add(*reinterpret_cast<const float2*>(rec), *reinterpret_cast<const float2*>(rec + 4 + 2 * (threadIdx.x & 31)));
  }
};

// The log-sum-exp of a unit of sequence b from its maximum and sum, the same in all lanes of the warp, and r = 1 / l
// (0 where no key has a share). A value that is not finite sets SISA_ST_NONFINITE, except where no key lies in a
// page of the pool: those table entries have set SISA_ST_BAD_POS, and nothing was read that could be at fault.
__device__ __forceinline__ float row_lse(const PagedAttnParams& p, int b, float m, float l, float& r) {
  const float lse = m + log2f(l);
  r = l == 0.f ? 0.f : 1.f / l;
  if (!isfinite(lse)) {
    const int lane = threadIdx.x & 31;
    bool any = l != 0.f;
    const int64_t pages = (keys_of(p, b) + (int64_t(1) << p.pg.page_shift) - 1) >> p.pg.page_shift;
    for (int64_t i = lane; i < pages && !any; i += 32)
      any = (unsigned)__ldg(p.pg.table + (int64_t)b * p.pg.table_sb + i) < (unsigned)p.pg.n_pages;
    if (__any_sync(0xffffffffu, any) && lane == 0 && p.status) atomicOr(p.status, SISA_ST_NONFINITE);
  }
  return lse;
}

// y and lse of unit bh = (b, h) from its complete sum.
template <bool kHalf>
__device__ __forceinline__ float write_row(const PagedAttnParams& p, int64_t bh, const Sum& s) {
  const int64_t b = bh / p.H, h = bh % p.H;
  const int lane = threadIdx.x & 31;
  float r;
  const float lse = row_lse(p, (int)b, s.m, s.l, r);
  reinterpret_cast<uint32_t*>(p.y + 2 * (b * p.y_sb + h * p.y_sh))[lane] = pack2<kHalf>(s.a.x * r, s.a.y * r);
  if (lane == 0 && p.lse_all) p.lse_all[bh] = lse;
  return lse;
}

// What a share's exponent is relative to: lse, or 0 where every score is -inf and no key has a share.
__device__ __forceinline__ float share_base(float lse) { return lse == -INFINITY ? 0.f : lse; }

// kUnit: a CTA has one unit to itself, its warps equal runs of that unit's tiles; y, lse and (from the scores
// kept in shared memory) the weights are finished here and no other kernel follows.
template <bool kHalf, bool kScores, bool kUnit>
__global__ void __launch_bounds__(NW * 32, 2) paged_attn_kernel(PagedAttnParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  if constexpr (!kUnit) asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t raw = smem_u32(smem_raw), sbase = (raw + 127u) & ~127u;
  uint8_t* gbase = smem_raw + (sbase - raw);
  const uint32_t ring = sbase + warp * SZ_WARP, bars = sbase + OFF_BAR + warp * NSTAGE * 8;
  uint8_t* gring = gbase + warp * SZ_WARP;
  uint32_t* masks = reinterpret_cast<uint32_t*>(gbase + OFF_MASK) + warp * NSTAGE;
  if (lane == 0) {
    for (int s = 0; s < NSTAGE; ++s) mbar_init(bars + 8 * s, 1);
    fence_barrier_init();
  }
  __syncwarp();

  // ---- this warp's run of tiles: count of them from cursor `in` on
  Cursor in{}, at;
  int64_t count = 0;
  if constexpr (kUnit) {
    in.b = blockIdx.x / p.H;
    in.h = blockIdx.x % p.H;
    in.load(p);
    in.t = in.T * warp / NW;
    count = in.T * (warp + 1) / NW - in.t;
    if (in.h == 0 && threadIdx.x == 0 && __ldg(p.lengths + in.b) > p.max_keys && p.status)
      atomicOr(p.status, SISA_ST_BAD_POS);
  } else {
    int64_t per_head;
    tiles_before(p, 0, per_head);
    const int64_t tiles = per_head * p.H, nwork = workers(tiles);
    if ((int64_t)blockIdx.x * NW >= nwork && blockIdx.x > 0) return;
    const int w = blockIdx.x * NW + warp;
    if (w == 0) {                               // lengths past the table, once per sequence
      for (int b = lane; b < p.B; b += 32)
        if (__ldg(p.lengths + b) > p.max_keys && p.status) atomicOr(p.status, SISA_ST_BAD_POS);
    }
    if (w < nwork) {
      const int64_t x0 = run_start(w, tiles);
      count = run_start(w + 1, tiles) - x0;
      in = find_tile(p, x0);
    }
  }
  at = in;
  // the pieces this warp leaves for the CTA's merge: [0] of the unit that began before its run (s_ends: and
  // ends in it), [1] of the one that goes on after it; s_unit -1: none
  __shared__ int64_t s_unit[NW][2];
  __shared__ bool s_ends[NW];
  __shared__ float s_lse;
  __shared__ float s_x[kScores && kUnit ? UNIT_KEYS : 1];
  float* pieces = reinterpret_cast<float*>(gbase + OFF_REC);
  if (lane == 0) { s_unit[warp][0] = s_unit[warp][1] = -1; s_ends[warp] = false; }
  __syncwarp();

  // ---- this lane's part of a tile's copies: operand op of the tile's sub-tile sub (pages of 16 slots
  // give a tile two sub-tiles)
  const int op = lane & 7, sub = lane >> 3;
  const int nsub = p.pg.page_shift < 5 ? 2 : 1, rows_max = p.pg.page_shift < 5 ? 16 : TK;
  const char* src0 = nullptr;
  int64_t src_p = 0, src_h = 0;                 // page and head strides in bytes
  int row_bytes = 0;
  uint32_t dst_off = 0;
  if (op == 0) { src0 = p.pg.k; src_p = p.pg.k_sp * 2; src_h = p.pg.k_sh * 2; row_bytes = 128; }
  if (op == 1) { src0 = p.pg.v; src_p = p.pg.v_sp * 2; src_h = p.pg.v_sh * 2; row_bytes = 128; dst_off = OFF_V; }
  if (op == 2) { src0 = p.pg.b; src_p = p.pg.b_sp * 2; src_h = p.pg.b_sh * 2; row_bytes = 64; dst_off = OFF_B; }
  if (op == 3) { src0 = (const char*)p.pg.g; src_p = p.pg.s_sp * 4; src_h = p.pg.s_sh * 4; row_bytes = 4; dst_off = OFF_G; }
  if (op == 4 && p.f_q) { src0 = (const char*)p.pg.f; src_p = p.pg.s_sp * 4; src_h = p.pg.s_sh * 4; row_bytes = 4; dst_off = OFF_F; }
  dst_off += sub * rows_max * row_bytes;
  const bool copier = sub < nsub && row_bytes > 0;
  const uint32_t key_bytes = 128 + 128 + 64 + 4 + (p.f_q ? 4 : 0);

  // the page of this lane's sub-tile at the fill cursor, read one tile ahead of its use
  auto page_at = [&]() {
    const int64_t j = in.t * TK + sub * rows_max;
    return sub < nsub && j < in.n ? __ldg(p.pg.table + (int64_t)in.b * p.pg.table_sb + (j >> p.pg.page_shift)) : -1;
  };
  int page = count > 0 ? page_at() : -1;
  int64_t filled = 0;
  const uint64_t policy = policy_evict_first();
  auto fill = [&](int s) {
    const int64_t j = in.t * TK + sub * rows_max;
    const int left = (int)(in.n - j < rows_max ? in.n - j : rows_max);       // keys of this sub-tile
    const bool used = sub < nsub && left > 0;
    const bool good = used && (unsigned)page < (unsigned)p.pg.n_pages;
    if (used && !good && op == 0 && p.status) atomicOr(p.status, SISA_ST_BAD_POS);
    const int rows = good ? (left + 3) & ~3 : 0;                             // copies are whole 16-byte units
    const uint32_t bits = good ? (left >= 32 ? 0xffffffffu : (1u << left) - 1) << (sub * rows_max) : 0u;
    const int rows1 = __shfl_sync(0xffffffffu, rows, 8);
    const uint32_t bits1 = __shfl_sync(0xffffffffu, bits, 8);
    if (lane == 0) {
      masks[s] = bits | bits1;
      mbar_expect_tx(bars + 8 * s, (uint32_t)(rows + rows1) * key_bytes);
    }
    __syncwarp();
    if (copier && rows > 0)
      bulk_load_hint(ring + s * SZ_STAGE + dst_off,
                     src0 + page * src_p + in.h * src_h + (j & ((1 << p.pg.page_shift) - 1)) * row_bytes,
                     (uint32_t)(rows * row_bytes), bars + 8 * s, policy);
    ++filled;
    if (filled < count) {
      in.next(p);
      page = page_at();
    }
  };
  for (int s = 0; s < NSTAGE && filled < count; ++s) fill(s);

  const int quad = lane >> 3, part = lane & 7;  // a lane holds 16 bytes (part) of key quad of every group
  const int key = 4 * part + quad;              // the key whose score this lane ends up with
  const float c1 = kScale * kLOG2E;
  float2 q2[4], c2[2], acc[4];
  float gq = 0.f, fq = 0.f, lam2 = 0.f, m_ref = -INFINITY, lsum = 0.f;
  int64_t seg = 0;                              // tiles of the unit done in this run
  bool ok = true;
#pragma unroll 1
  for (int64_t i = 0; i < count; ++i) {
    if (seg == 0) {                             // a new unit: its query row and constants
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.q + 2 * (at.b * p.q_sb + at.h * p.q_sh)) + part);
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p.c + 2 * (at.b * p.c_sb + at.h * p.c_sh)) + part);
      q2[0] = unpack2<kHalf>(v.x); q2[1] = unpack2<kHalf>(v.y); q2[2] = unpack2<kHalf>(v.z); q2[3] = unpack2<kHalf>(v.w);
      c2[0] = unpack2<kHalf>(u.x); c2[1] = unpack2<kHalf>(u.y);
      const int64_t bh = (int64_t)at.b * p.H + at.h;
      gq = __ldg(p.g_q + bh);
      fq = p.f_q ? __ldg(p.f_q + bh) : 0.f;
      lam2 = __ldg(p.lam + at.h) * kLOG2E;
      m_ref = -INFINITY;
      lsum = 0.f;
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[d] = bcast2(0.f);
    }
    const int s = (int)(i % NSTAGE);
    if (!warp_wait_tested<true>(bars + 8 * s, (uint32_t)(i / NSTAGE) & 1, p.status)) { ok = false; break; }
    const uint8_t* st = gring + s * SZ_STAGE;
    const uint32_t mask = masks[s];
    float qk[8], cb[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint4 kv = reinterpret_cast<const uint4*>(st)[e * 32 + lane];
      const uint2 bv = reinterpret_cast<const uint2*>(st + OFF_B)[e * 32 + lane];
      float2 a = mul2(q2[0], unpack2<kHalf>(kv.x)), d = mul2(c2[0], unpack2<kHalf>(bv.x));
      a = fma2(q2[1], unpack2<kHalf>(kv.y), a);
      a = fma2(q2[2], unpack2<kHalf>(kv.z), a);
      a = fma2(q2[3], unpack2<kHalf>(kv.w), a);
      d = fma2(c2[1], unpack2<kHalf>(bv.y), d);
      qk[e] = a.x + a.y;
      cb[e] = d.x + d.y;
    }
    const float gj = reinterpret_cast<const float*>(st + OFF_G)[key];
    const float fj = p.f_q ? reinterpret_cast<const float*>(st + OFF_F)[key] : 0.f;
    const float dec = ex2_approx(fmin_nan((gq - gj) * kLOG2E, 0.f));
    float x = fmaf(reduce_scatter8(qk, part), c1, lam2 * (dec * reduce_scatter8(cb, part)));
    x = (mask >> key) & 1 ? fmaf(fq - fj, kLOG2E, x) : -INFINITY;
    if constexpr (kScores) {
      const int64_t j = at.t * TK + key;
      if (kUnit) s_x[j] = x;
      else if (j < at.n) p.scores[((int64_t)at.b * p.H + at.h) * p.max_keys + j] = x;
    }
    if (__any_sync(0xffffffffu, x > m_ref + 8.f)) {
      float mx = x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float corr = (m_ref == -INFINITY) ? 0.f : exp2f(m_ref - mx);
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[d] = mul2(acc[d], bcast2(corr));
      lsum *= corr;
      m_ref = mx;
    }
    const float pj = ex2_approx(x - (m_ref == -INFINITY ? 0.f : m_ref));   // below 2^-126: 0
    lsum += pj;
    if (mask == 0xffffffffu) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 pe = bcast2(__shfl_sync(0xffffffffu, pj, (lane & 24) + e));
        const uint4 v = reinterpret_cast<const uint4*>(st + OFF_V)[e * 32 + lane];
        acc[0] = fma2(pe, unpack2<kHalf>(v.x), acc[0]);
        acc[1] = fma2(pe, unpack2<kHalf>(v.y), acc[1]);
        acc[2] = fma2(pe, unpack2<kHalf>(v.z), acc[2]);
        acc[3] = fma2(pe, unpack2<kHalf>(v.w), acc[3]);
      }
    } else {
      // a partial tile: whatever lies in the slots past the end (NaN too) must not meet the sums
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        const float2 pe = bcast2(__shfl_sync(0xffffffffu, pj, (lane & 24) + e));
        uint4 v = make_uint4(0, 0, 0, 0);
        if ((mask >> (4 * e + quad)) & 1) v = reinterpret_cast<const uint4*>(st + OFF_V)[e * 32 + lane];
        acc[0] = fma2(pe, unpack2<kHalf>(v.x), acc[0]);
        acc[1] = fma2(pe, unpack2<kHalf>(v.y), acc[1]);
        acc[2] = fma2(pe, unpack2<kHalf>(v.z), acc[2]);
        acc[3] = fma2(pe, unpack2<kHalf>(v.w), acc[3]);
      }
    }
    __syncwarp();                               // every lane has read the stage
    if (filled < count) fill(s);
    ++seg;
    if (at.t + 1 == at.T || i + 1 == count) {
      // ---- the unit ends here, or the run does: this run's m, l and 64 sums
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        acc[d].x += __shfl_xor_sync(0xffffffffu, acc[d].x, 8);
        acc[d].y += __shfl_xor_sync(0xffffffffu, acc[d].y, 8);
        acc[d].x += __shfl_xor_sync(0xffffffffu, acc[d].x, 16);
        acc[d].y += __shfl_xor_sync(0xffffffffu, acc[d].y, 16);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, o);
      const int64_t bh = (int64_t)at.b * p.H + at.h;
      if (seg == at.T) {                        // the whole unit
        float r;
        const float lse = row_lse(p, at.b, m_ref, lsum, r);
        if (quad == 0) {
          const uint4 o = make_uint4(pack2<kHalf>(acc[0].x * r, acc[0].y * r), pack2<kHalf>(acc[1].x * r, acc[1].y * r),
                                     pack2<kHalf>(acc[2].x * r, acc[2].y * r), pack2<kHalf>(acc[3].x * r, acc[3].y * r));
          reinterpret_cast<uint4*>(p.y + 2 * (at.b * p.y_sb + at.h * p.y_sh))[part] = o;
        }
        if (lane == 0) {
          if (kUnit) s_lse = lse;
          if (!kUnit || p.lse_all) p.lse_all[bh] = lse;
        }
      } else {
        const int kind = at.t + 1 == seg ? 1 : 0;
        float* rec = pieces + (warp * 2 + kind) * REC;
        if (lane == 0) {
          *reinterpret_cast<float2*>(rec) = make_float2(m_ref, lsum);
          s_unit[warp][kind] = bh;
          if (kind == 0) s_ends[warp] = at.t + 1 == at.T;
        }
        if (quad == 0) {
          reinterpret_cast<float4*>(rec + 4)[2 * part] = make_float4(acc[0].x, acc[0].y, acc[1].x, acc[1].y);
          reinterpret_cast<float4*>(rec + 4)[2 * part + 1] = make_float4(acc[2].x, acc[2].y, acc[3].x, acc[3].y);
        }
      }
      seg = 0;
    }
    if (i + 1 < count) at.next(p);
  }
  if (!ok) {                                    // a wait ran out: let the copies in flight land before leaving
    for (int s = 0; s < NSTAGE && s < filled; ++s)
      mbar_wait<true>(bars + 8 * s, (uint32_t)((filled - 1 - s) / NSTAGE) & 1, p.status);
  }
  // ---- the CTA's runs are neighbours: one warp merges their pieces in order. What began before the CTA or
  // goes on after it becomes its record 0 or 1.
  __syncthreads();
  if (!kUnit && warp != 0) return;
  Sum sum;
  int64_t unit = -1;                            // the unit being merged, -1: none
  bool before = false;                          // it began before this CTA
  auto close = [&](bool ends) {
    if (ends && !before) {
      const float lse = write_row<kHalf>(p, unit, sum);
      if (kUnit && lane == 0) s_lse = lse;
    } else if (!kUnit) {                        // (a unit's own CTA leaves pieces only when a wait ran out)
      float* rec = p.records + ((int64_t)blockIdx.x * 2 + (before ? 0 : 1)) * REC;
      if (lane == 0) *reinterpret_cast<float2*>(rec) = make_float2(sum.m, sum.l);
      *reinterpret_cast<float2*>(rec + 4 + 2 * lane) = sum.a;
    }
    unit = -1;
  };
#pragma unroll 1
  for (int i = 0; i < NW && warp == 0; ++i) {
    if (s_unit[i][0] >= 0) {
      if (unit < 0) { unit = s_unit[i][0]; before = true; sum.clear(); }
      sum.add(pieces + (i * 2) * REC);
      if (s_ends[i]) close(true);
    }
    if (s_unit[i][1] >= 0) {
      unit = s_unit[i][1];
      before = false;
      sum.clear();
      sum.add(pieces + (i * 2 + 1) * REC);
    }
  }
  if (unit >= 0) close(false);
  if constexpr (kUnit) {
    const int64_t b = blockIdx.x / p.H, h = blockIdx.x % p.H, n = keys_of(p, (int)b);
    if (n == 0 && warp == 0) {                  // a row with no keys
      reinterpret_cast<uint32_t*>(p.y + 2 * (b * p.y_sb + h * p.y_sh))[lane] = 0u;
      if (lane == 0 && p.lse_all) p.lse_all[blockIdx.x] = -INFINITY;
    }
    if constexpr (kScores) {
      __syncthreads();
      const float lse = share_base(s_lse);
      for (int64_t j = threadIdx.x; j < n; j += NW * 32) {
        const int page = page_of(p.pg, (int)b, j, nullptr);
        if (page < 0) continue;
        const int64_t slot = page * p.pg.s_sp + h * p.pg.s_sh + (j & ((1 << p.pg.page_shift) - 1));
        p.weight_out[slot] = p.pg.weight[slot] + ex2_approx(s_x[j] - lse);
      }
    }
  }
}

constexpr int JW = 8;
// The CTAs that hold pieces of unit (b, h), found by warp 0 from the lengths alone, then (every thread) the end
// of the kernel that writes the records.
__device__ __forceinline__ int2 unit_span(const PagedAttnParams& p, int b, int h, int64_t n) {
  __shared__ int s_span[2];
  if (threadIdx.x < 32) {
    int64_t all;
    const int64_t T = (n + TK - 1) / TK, u0 = tiles_before(p, b, all) * p.H + h * T, tiles = all * p.H;
    if (threadIdx.x == 0) {
      s_span[0] = T == 0 ? 0 : worker_of(u0, tiles) / NW;
      s_span[1] = T == 0 ? 0 : worker_of(u0 + T - 1, tiles) / NW;
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __syncthreads();
  return make_int2(s_span[0], s_span[1]);
}

// The records of one unit, merged by the JW warps of a block: each takes a run of them (the maximum first,
// then every record on its own, so that the loads are in flight together), and warp 0 the runs' sums, all in
// CTA order. Returns false (to every warp) for a unit that one CTA finished or that has no keys; the sum is
// warp 0's.
__device__ __forceinline__ bool join_unit(const PagedAttnParams& p, int2 span, Sum& sum) {
  const int c0 = span.x, c1 = span.y;
  if (c0 == c1) return false;
  __shared__ __align__(16) float s_sum[JW][REC];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (c1 - c0 + JW) / JW, lo = c0 + warp * per, hi = min(c1 + 1, lo + per);
  auto rec = [&](int c) { return p.records + ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * REC; };
  sum.clear();
  for (int c = lo; c < hi; c += 32) {
    const float2 ml = c + lane < hi ? *reinterpret_cast<const float2*>(rec(c + lane)) : make_float2(-INFINITY, 0.f);
    float m = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float sc = exp2f(ml.x - (m == -INFINITY ? 0.f : m));
    float l = ml.y * sc;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float2 a = bcast2(0.f);
    const int cnt = min(32, hi - c);
#pragma unroll 8
    for (int i = 0; i < cnt; ++i)
      a = fma2(*reinterpret_cast<const float2*>(rec(c + i) + 4 + 2 * lane), bcast2(__shfl_sync(0xffffffffu, sc, i)), a);
    sum.add(make_float2(m, l), a);
  }
  if (lane == 0) *reinterpret_cast<float2*>(s_sum[warp]) = make_float2(sum.m, sum.l);
  *reinterpret_cast<float2*>(s_sum[warp] + 4 + 2 * lane) = sum.a;
  __syncthreads();
  if (warp == 0)
    for (int i = 1; i < JW; ++i) sum.add(s_sum[i]);
  return true;
}

// y and lse of a unit that several CTAs share, or of a row with no keys, by one warp.
template <bool kHalf>
__device__ __forceinline__ void finish_unit(const PagedAttnParams& p, int64_t bh, int64_t n, bool joined, const Sum& sum) {
  const int64_t b = bh / p.H, h = bh % p.H;
  const int lane = threadIdx.x & 31;
  if (joined) {
    write_row<kHalf>(p, bh, sum);
  } else if (n == 0) {
    reinterpret_cast<uint32_t*>(p.y + 2 * (b * p.y_sb + h * p.y_sh))[lane] = 0u;
    if (lane == 0) p.lse_all[bh] = -INFINITY;
  }
}

template <bool kHalf>
__global__ void __launch_bounds__(JW * 32) paged_join_kernel(PagedAttnParams p) {
  const int64_t bh = blockIdx.x;
  const int64_t n = keys_of(p, (int)(bh / p.H));
  Sum sum;
  const bool joined = join_unit(p, unit_span(p, (int)(bh / p.H), (int)(bh % p.H), n), sum);
  if (threadIdx.x < 32) finish_unit<kHalf>(p, bh, n, joined, sum);
}

// weight_out_j = weight_j + 2^(x_j - lse), four keys per thread and step (a page holds a multiple of four).
// A unit has gridDim.x blocks, each with every gridDim.x-th run of 1024 keys; the first one also finishes the
// unit. The loads of a block's first step do not need lse and are issued ahead of the join.
constexpr int WT = JW * 32;
template <bool kHalf>
__global__ void __launch_bounds__(WT) paged_weights_kernel(PagedAttnParams p) {
  const int64_t bh = blockIdx.y;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int64_t n = keys_of(p, b), step = (int64_t)gridDim.x * WT * 4;
  if (blockIdx.x > 0 && (int64_t)blockIdx.x * WT * 4 >= n) return;
  const float* xs = p.scores + bh * p.max_keys;
  struct Four { int64_t at; float4 x, w; };      // at < 0: nothing to do
  auto place = [&](int64_t j) -> int64_t {
    if (j >= n) return -1;
    const int page = page_of(p.pg, b, j, nullptr);
    return page < 0 ? -1 : page * p.pg.s_sp + h * p.pg.s_sh + (j & ((1 << p.pg.page_shift) - 1));
  };
  int64_t j = (int64_t)blockIdx.x * WT * 4 + threadIdx.x * 4;
  // the last four of a unit may reach past its end: those slots are the page's own and are not stored
  Four f;
  f.at = place(j);
  f.w = f.at >= 0 ? *reinterpret_cast<const float4*>(p.pg.weight + f.at) : make_float4(0.f, 0.f, 0.f, 0.f);
  const int2 span = unit_span(p, b, h, n);
  f.x = f.at >= 0 ? *reinterpret_cast<const float4*>(xs + j) : make_float4(0.f, 0.f, 0.f, 0.f);
  __shared__ float s_lse;
  Sum sum;
  const bool joined = join_unit(p, span, sum);
  if (threadIdx.x < 32) {
    if (blockIdx.x == 0) finish_unit<kHalf>(p, bh, n, joined, sum);
    if (threadIdx.x == 0 && n > 0) s_lse = joined ? sum.m + log2f(sum.l) : p.lse_all[bh];
  }
  __syncthreads();
  const float lse = share_base(s_lse);
  for (; j - threadIdx.x * 4 < n; j += step) {
    Four g;
    g.at = place(j + step);
    if (g.at >= 0) {
      g.w = *reinterpret_cast<const float4*>(p.pg.weight + g.at);
      g.x = *reinterpret_cast<const float4*>(xs + j + step);
    }
    if (f.at >= 0) {
      f.w.x += ex2_approx(f.x.x - lse); f.w.y += ex2_approx(f.x.y - lse);
      f.w.z += ex2_approx(f.x.z - lse); f.w.w += ex2_approx(f.x.w - lse);
      float* out = p.weight_out + f.at;
      if (j + 4 <= n) {
        *reinterpret_cast<float4*>(out) = f.w;
      } else {
        out[0] = f.w.x;
        if (j + 1 < n) out[1] = f.w.y;
        if (j + 2 < n) out[2] = f.w.z;
      }
    }
    f = g;
  }
}

// A kernel launched so that its blocks may be resident before the previous kernel of the stream ends
// (they wait for it themselves).
template <typename K>
cudaError_t launch_after(K kernel, dim3 grid, int threads, cudaStream_t st, const PagedAttnParams& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <bool kHalf>
cudaError_t launch(const PagedAttnParams& p, cudaStream_t st) {
  // Short tables: one launch and no join. 16 heads, one CTA per unit against the split (us in a captured graph, L2
  // flushed before each, without / with weights): 256 keys, 1 x 12.2 / 12.3 against 14.4 / 15.3, 16 x 14.4 / 16.4
  // against 18.5 / 20.5, 64 x 32.8 / 37.0 against 30.6 / 33.8; 512 keys, 1 x 14.3 / 16.4 against 14.3 / 14.4, 16 x
  // 18.4 / 20.5 against 22.6 / 22.6, 32 x 28.7 / 32.8 against 28.7 / 30.7, 64 x 47.1 / 55.3 against 43.0 / 47.1; 1024
  // keys, 1 x 18.4 / 21.3 against 15.4 / 17.5. So it pays up to about 256 units and costs up to 8 us at 1024 units.
  // The rule sees the table, not the lengths: 77 keys x 8 heads take 10.2 under a table of 512 and 14.4 under one of 4096.
  const bool unit = p.max_keys <= UNIT_KEYS;
  auto* main = p.weight_out ? (unit ? paged_attn_kernel<kHalf, true, true> : paged_attn_kernel<kHalf, true, false>)
                            : (unit ? paged_attn_kernel<kHalf, false, true> : paged_attn_kernel<kHalf, false, false>);
  cudaError_t e = cudaFuncSetAttribute(main, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
  if (e != cudaSuccess) return e;
  if (unit) {
    main<<<p.B * p.H, NW * 32, SMEM_BYTES, st>>>(p);
    return cudaGetLastError();
  }
  // As many CTAs as the table could need (workers() never falls with the tiles): the lengths are only known on
  // the device, and every CTA without work still costs its launch.
  const int64_t most = workers((int64_t)p.B * p.H * ((p.max_keys + TK - 1) / TK));
  main<<<(unsigned)((most + NW - 1) / NW), NW * 32, SMEM_BYTES, st>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int units = p.B * p.H;
  if (!p.weight_out) return launch_after(paged_join_kernel<kHalf>, dim3(units), JW * 32, st, p);
  // about eight blocks per SM over all units, at most one per run of 1024 keys
  const int64_t runs = (p.max_keys + WT * 4 - 1) / (WT * 4), want = (148 * 8 + units - 1) / units;
  return launch_after(paged_weights_kernel<kHalf>, dim3((unsigned)(want < runs ? want : runs), units), WT, st, p);
}

}  // namespace pat

int64_t paged_attn_workspace_floats(int64_t units, int64_t max_keys, bool scores) {
  if (max_keys <= pat::UNIT_KEYS) return 0;      // one CTA per unit: nothing passes between kernels
  const int64_t base = (int64_t)pat::NCTA * 2 * pat::REC + ((units + 3) & ~int64_t(3));
  return base + (scores ? units * max_keys : 0);
}

cudaError_t launch_paged_attn(PagedAttnParams p, int dtype, cudaStream_t st) {
  const int64_t units = (int64_t)p.B * p.H;
  p.lse_all = p.lse;
  if (p.ws) {
    p.records = p.ws;
    if (!p.lse) p.lse_all = p.ws + (int64_t)pat::NCTA * 2 * pat::REC;
    p.scores = p.ws + paged_attn_workspace_floats(units, p.max_keys, false);
  }
  return dtype == 1 ? pat::launch<true>(p, st) : pat::launch<false>(p, st);
}

}  // namespace sisa
