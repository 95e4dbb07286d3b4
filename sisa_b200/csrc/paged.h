// Host-side launch parameters of the paged-cache kernels (paged_attn.cu, paged_cache.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

#include "sisa_b200.h"

namespace sisa {

// The pages as the kernels address them: k, v, b~ rows in 16-bit elements (a page's rows of one head are
// dense), one fp32 / int32 plane element per slot; strides in elements.
struct PageView {
  char* k; char* v; char* b;
  float* g; float* f; float* weight; int32_t* token;
  int64_t k_sp, k_sh, v_sp, v_sh, b_sp, b_sh, s_sp, s_sh;
  int n_pages, page_shift;               // page_size = 1 << page_shift
  const int32_t* table;                  // (B, max_pages) page of each sequence's block of slots
  int64_t table_sb;
  int max_pages;
};

struct PagedAttnParams {
  PageView pg;
  const char* q; int64_t q_sb, q_sh;     // (B, H, 1, 64) low precision
  const char* c; int64_t c_sb, c_sh;     // (B, H, 1, 32)
  const float* g_q;                      // (B, H)
  const float* f_q;                      // (B, H) or null (then pg.f is not read)
  const int32_t* lengths;                // (B,) keys of each sequence; 0 for an idle row
  const float* lam;
  char* y; int64_t y_sb, y_sh;           // (B, H, 1, 64) low precision
  float* lse;                            // (B, H) log2 units, or null
  float* weight_out;                     // null: weights are not accumulated
  float* ws;                             // the workspace; its parts are set by launch_paged_attn:
  float* records; float* lse_all; float* scores;
  int B, H;
  int64_t max_keys;                      // max_pages << page_shift
  int32_t* status;
};

struct PagedEvictParams {
  PageView pg;
  const int32_t* position;               // (B,) index of the incoming token, < 0 for an idle row
  int B, H;
  int64_t budget, recent;
  int32_t* slots;                        // (B, H)
  int32_t* status;
};

struct PagedAppendParams {
  PageView pg;
  const uint16_t* proj; int64_t proj_sb;
  const float* z; int64_t z_sb;          // (B, H) forget logits or null
  int col_k, col_v, col_b, col_c, col_th, col_a;
  const int32_t* position;
  const int32_t* slots;                  // (B, H) or null; entries < 0 take the position
  int64_t cap;                           // slots must lie in [0, cap)
  int64_t budget;                        // lengths are min(position + 1, budget); 0: position + 1
  const float* carry_in; float* carry_out;   // (B, H, 18): phi 0..15, g, F; may be the same
  uint16_t* c_out; float* g_out; float* f_out;
  int32_t* lengths;                      // (B,) or null
  int B, H;
  int32_t* status;
};

struct PagedFillParams {
  PageView pg;
  const char* k; int64_t k_sb, k_sh, k_sl;   // (B, H, L, 64) views, low precision
  const char* v; int64_t v_sb, v_sh, v_sl;
  const char* b; int64_t b_sb, b_sh, b_sl;   // (B, H, L, 32)
  const float* g; const float* f;        // (B, H, L) unit stride along L; f null: zeros are written
  int64_t g_sb, g_sh, f_sb, f_sh;
  const float* weight;                   // (B, H, L) contiguous or null (then keep == L)
  int64_t L, keep, recent;
  int32_t* index;                        // workspace (B, H, keep)
  int B, H;
  int32_t* status;
};

int64_t paged_attn_workspace_floats(int64_t units, int64_t max_keys, bool scores);
cudaError_t launch_paged_attn(PagedAttnParams p, int dtype, cudaStream_t st);
cudaError_t launch_paged_evict(const PagedEvictParams& p, cudaStream_t st);
cudaError_t launch_paged_append(const PagedAppendParams& p, int dtype, cudaStream_t st);
cudaError_t launch_paged_fill(PagedFillParams p, cudaStream_t st);

// The page that holds slots [j, ...) of sequence b, or -1 (and SISA_ST_BAD_POS) if the table's entry names
// no page of the pool.
__device__ __forceinline__ int page_of(const PageView& pg, int b, int64_t j, int32_t* status) {
  const int page = __ldg(pg.table + (int64_t)b * pg.table_sb + (j >> pg.page_shift));
  if ((unsigned)page < (unsigned)pg.n_pages) return page;
  if (status) atomicOr(status, SISA_ST_BAD_POS);
  return -1;
}

// An fp32 weight as an unsigned integer in the same order: NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

}  // namespace sisa
