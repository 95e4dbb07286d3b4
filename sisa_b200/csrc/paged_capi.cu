// paged_capi.cu - the extern "C" entry points of the paged cache: argument checks and launches. No device
// allocation, no host synchronisation, no exceptions. Every call makes the device that owns the pages current
// while it launches: the stream handle 0 names the current device's default stream, and a kernel launched on
// another GPU would run there with these addresses.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>

#include "sisa_b200.h"
#include "paged.h"
#include "capi_util.h"

using sisa::capi_fail;

namespace {

int fail(int code, const char* what, const char* msg) {
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, msg);
  return capi_fail(code, buf);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The pages, their block table and the sizes that every entry point shares.
int make_view(sisa::PageView& o, const sisa_pages* pg, const int32_t* table, int64_t table_sb, int64_t max_pages,
              int64_t B, int64_t H, bool rows, const char* what) {
  if (B < 1 || H < 1 || B > 65535 || H > 65535 || B * H > 65535)
    return fail(SISA_ERR_VALUE, what, "B and H must be >= 1 with B*H <= 65535");
  if (!pg || !table) return fail(SISA_ERR_VALUE, what, "null pages or block table");
  int shift = 4;
  while (shift <= 8 && (int64_t(1) << shift) != pg->page_size) ++shift;
  if (shift > 8) return fail(SISA_ERR_VALUE, what, "page_size must be 16, 32, 64, 128 or 256");
  if (pg->n_pages < 1 || pg->n_pages > (int64_t(1) << 30) || max_pages < 1 || max_pages > (int64_t(1) << 22))
    return fail(SISA_ERR_VALUE, what, "n_pages outside [1, 2^30] or max_pages outside [1, 2^22]");
  if (!aligned(table, 4) || table_sb < max_pages)
    return fail(SISA_ERR_VALUE, what, "block table must be 4-byte aligned with rows of max_pages entries");
  if (rows) {
    if (!pg->k || !pg->v || !pg->b || !pg->g) return fail(SISA_ERR_VALUE, what, "null k, v, b or g pages");
    if (!aligned(pg->k, 16) || !aligned(pg->v, 16) || !aligned(pg->b, 16))
      return fail(SISA_ERR_ALIGN, what, "k, v and b pages must be 16-byte aligned");
    if ((pg->k_sp | pg->k_sh | pg->v_sp | pg->v_sh | pg->b_sp | pg->b_sh) % 8)
      return fail(SISA_ERR_ALIGN, what, "page and head strides of k, v and b must be multiples of 8 elements");
    if (pg->k_sh < 64 * pg->page_size || pg->v_sh < 64 * pg->page_size || pg->b_sh < 32 * pg->page_size)
      return fail(SISA_ERR_VALUE, what, "a head's rows of k, v and b must be dense within a page");
    if (pg->k_sp < 0 || pg->v_sp < 0 || pg->b_sp < 0) return fail(SISA_ERR_VALUE, what, "negative page strides");
  }
  if (!aligned(pg->g, 16) || !aligned(pg->f, 16) || !aligned(pg->weight, 16) || !aligned(pg->token, 16) ||
      (pg->s_sp | pg->s_sh) % 4)
    return fail(SISA_ERR_ALIGN, what, "the g, f, weight and token planes must be 16-byte aligned, strides in 4 elements");
  if (pg->s_sh < pg->page_size || pg->s_sp < 0)
    return fail(SISA_ERR_VALUE, what, "a head's plane values must be dense within a page");
  o.k = static_cast<char*>(pg->k); o.v = static_cast<char*>(pg->v); o.b = static_cast<char*>(pg->b);
  o.g = pg->g; o.f = pg->f; o.weight = pg->weight; o.token = pg->token;
  o.k_sp = pg->k_sp; o.k_sh = pg->k_sh; o.v_sp = pg->v_sp; o.v_sh = pg->v_sh; o.b_sp = pg->b_sp; o.b_sh = pg->b_sh;
  o.s_sp = pg->s_sp; o.s_sh = pg->s_sh;
  o.n_pages = (int)pg->n_pages; o.page_shift = shift;
  o.table = table; o.table_sb = table_sb; o.max_pages = (int)max_pages;
  return SISA_OK;
}

int launched(cudaError_t e, const char* what) {
  return e == cudaSuccess ? SISA_OK : fail(SISA_ERR_CUDA, what, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int64_t sisa_paged_attn_workspace(int64_t B, int64_t H, int64_t max_keys, int accumulate) {
  return 4 * sisa::paged_attn_workspace_floats(B * H, max_keys, accumulate != 0);
}

int sisa_paged_attn(const sisa_view4* q, const sisa_view4* c, const float* g_q, const float* f_q,
                    const sisa_pages* pages, const int32_t* table, int64_t table_sb, int64_t max_pages,
                    const int32_t* lengths, const float* lam, int64_t B, int64_t H, int dtype, const sisa_view4* y,
                    float* lse, float* weight_out, void* workspace, int32_t* status, void* stream) {
  const char* what = "sisa_paged_attn";
  sisa::PagedAttnParams p{};
  int rc;
  if ((rc = sisa::capi_check_dtype(dtype))) return rc;
  if ((rc = make_view(p.pg, pages, table, table_sb, max_pages, B, H, true, what))) return rc;
  if ((rc = sisa::capi_check_view(q, 2, "q")) || (rc = sisa::capi_check_view(c, 2, "c")) ||
      (rc = sisa::capi_check_view(y, 2, "y")))
    return rc;
  const int64_t max_keys = max_pages * pages->page_size;
  if (!g_q || !lengths || !lam) return fail(SISA_ERR_VALUE, what, "null pointer");
  const bool needs_ws = sisa::paged_attn_workspace_floats(B * H, max_keys, false) > 0;
  if (needs_ws && !workspace) return fail(SISA_ERR_VALUE, what, "null workspace");
  if (f_q && !pages->f) return fail(SISA_ERR_VALUE, what, "f_q is given but the pages hold no f");
  if (weight_out && !pages->weight) return fail(SISA_ERR_VALUE, what, "weight_out is given but the pages hold no weight");
  if (!aligned(workspace, 16) || !aligned(weight_out, 16))
    return fail(SISA_ERR_ALIGN, what, "workspace and weight_out must be 16-byte aligned");
  sisa::DeviceScope scope;
  if ((rc = scope.bind(pages->k))) return rc;
  p.q = static_cast<const char*>(q->data); p.q_sb = q->stride_b; p.q_sh = q->stride_h;
  p.c = static_cast<const char*>(c->data); p.c_sb = c->stride_b; p.c_sh = c->stride_h;
  p.g_q = g_q; p.f_q = f_q; p.lengths = lengths; p.lam = lam;
  p.y = static_cast<char*>(y->data); p.y_sb = y->stride_b; p.y_sh = y->stride_h;
  p.lse = lse; p.weight_out = weight_out; p.ws = needs_ws ? static_cast<float*>(workspace) : nullptr;
  p.B = (int)B; p.H = (int)H; p.max_keys = max_keys;
  p.status = status;
  return launched(sisa::launch_paged_attn(p, dtype, static_cast<cudaStream_t>(stream)), what);
}

int sisa_paged_evict(const sisa_pages* pages, const int32_t* table, int64_t table_sb, int64_t max_pages,
                     const int32_t* position, int64_t B, int64_t H, int64_t budget, int64_t recent, int32_t* slots,
                     int32_t* status, void* stream) {
  const char* what = "sisa_paged_evict";
  sisa::PagedEvictParams p{};
  int rc;
  if ((rc = make_view(p.pg, pages, table, table_sb, max_pages, B, H, false, what))) return rc;
  if (!position || !slots) return fail(SISA_ERR_VALUE, what, "null pointer");
  if (!pages->weight || !pages->token) return fail(SISA_ERR_VALUE, what, "the pages hold no weight or token plane");
  if (budget < 1 || budget > max_pages * pages->page_size)
    return fail(SISA_ERR_VALUE, what, "budget outside [1, max_pages * page_size]");
  if (recent < 0 || recent >= budget) return fail(SISA_ERR_VALUE, what, "recent outside [0, budget)");
  sisa::DeviceScope scope;
  if ((rc = scope.bind(pages->weight))) return rc;
  p.position = position; p.B = (int)B; p.H = (int)H; p.budget = budget; p.recent = recent; p.slots = slots;
  p.status = status;
  return launched(sisa::launch_paged_evict(p, static_cast<cudaStream_t>(stream)), what);
}

int sisa_paged_append(const void* proj, int64_t proj_sb, const float* z, int64_t z_sb, const sisa_pages* pages,
                      const int32_t* table, int64_t table_sb, int64_t max_pages, const int32_t* position,
                      const int32_t* slots, int64_t budget, int64_t B, int64_t H, int dtype, const float* carry_in,
                      float* carry_out, void* c_out, float* g_out, float* f_out, int32_t* lengths, int32_t* status,
                      void* stream) {
  const char* what = "sisa_paged_append";
  sisa::PagedAppendParams p{};
  int rc;
  if ((rc = sisa::capi_check_dtype(dtype))) return rc;
  if ((rc = make_view(p.pg, pages, table, table_sb, max_pages, B, H, true, what))) return rc;
  if (!proj || !position || !carry_in || !carry_out || !c_out || !g_out) return fail(SISA_ERR_VALUE, what, "null pointer");
  if ((z == nullptr) != (f_out == nullptr)) return fail(SISA_ERR_VALUE, what, "z and f_out must both be given or both be null");
  if (z && !pages->f) return fail(SISA_ERR_VALUE, what, "z is given but the pages hold no f");
  const int64_t cap = max_pages * pages->page_size;
  if (budget < 0 || budget > cap) return fail(SISA_ERR_VALUE, what, "budget outside [0, max_pages * page_size]");
  int64_t off[9];
  if ((rc = sisa_fused_layout(H, off))) return rc;
  if (!aligned(proj, 4) || proj_sb < off[7] || proj_sb % 2 || !aligned(c_out, 4))
    return fail(SISA_ERR_ALIGN, what, "proj rows must hold 273 H elements, 4-byte aligned with an even stride");
  sisa::DeviceScope scope;
  if ((rc = scope.bind(pages->k))) return rc;
  p.proj = static_cast<const uint16_t*>(proj); p.proj_sb = proj_sb; p.z = z; p.z_sb = z_sb;
  p.col_k = (int)off[1]; p.col_v = (int)off[2]; p.col_b = (int)off[3]; p.col_c = (int)off[4];
  p.col_th = (int)off[5]; p.col_a = (int)off[6];
  p.position = position; p.slots = slots; p.budget = budget; p.cap = budget > 0 ? budget : cap;
  p.carry_in = carry_in; p.carry_out = carry_out; p.c_out = static_cast<uint16_t*>(c_out);
  p.g_out = g_out; p.f_out = f_out; p.lengths = lengths; p.B = (int)B; p.H = (int)H; p.status = status;
  return launched(sisa::launch_paged_append(p, dtype, static_cast<cudaStream_t>(stream)), what);
}

int64_t sisa_paged_fill_workspace(int64_t B, int64_t H, int64_t keep) { return 4 * B * H * keep; }

int sisa_paged_fill(const sisa_pages* pages, const int32_t* table, int64_t table_sb, int64_t max_pages,
                    const sisa_view4* k, const sisa_view4* v, const sisa_view4* b, const float* g, int64_t g_sb,
                    int64_t g_sh, const float* f, int64_t f_sb, int64_t f_sh, const float* weight, int64_t B, int64_t H,
                    int64_t L, int64_t keep, int64_t recent, void* workspace, int32_t* status, void* stream) {
  const char* what = "sisa_paged_fill";
  sisa::PagedFillParams p{};
  int rc;
  if ((rc = sisa::capi_check_dims(B, H, L))) return rc;
  if ((rc = make_view(p.pg, pages, table, table_sb, max_pages, B, H, true, what))) return rc;
  if ((rc = sisa::capi_check_view(k, 2, "k")) || (rc = sisa::capi_check_view(v, 2, "v")) ||
      (rc = sisa::capi_check_view(b, 2, "b")))
    return rc;
  if (!g || !workspace) return fail(SISA_ERR_VALUE, what, "null pointer");
  if (f && !pages->f) return fail(SISA_ERR_VALUE, what, "f is given but the pages hold no f");
  if (keep < 1 || keep > L || keep > max_pages * pages->page_size)
    return fail(SISA_ERR_VALUE, what, "keep outside [1, min(L, max_pages * page_size)]");
  if (recent < 0 || recent > keep) return fail(SISA_ERR_VALUE, what, "recent outside [0, keep]");
  if (!weight && keep != L) return fail(SISA_ERR_VALUE, what, "keeping fewer than L keys needs their weights");
  if (!aligned(workspace, 16)) return fail(SISA_ERR_ALIGN, what, "workspace must be 16-byte aligned");
  sisa::DeviceScope scope;
  if ((rc = scope.bind(pages->k))) return rc;
  p.k = static_cast<const char*>(k->data); p.k_sb = k->stride_b; p.k_sh = k->stride_h; p.k_sl = k->stride_l;
  p.v = static_cast<const char*>(v->data); p.v_sb = v->stride_b; p.v_sh = v->stride_h; p.v_sl = v->stride_l;
  p.b = static_cast<const char*>(b->data); p.b_sb = b->stride_b; p.b_sh = b->stride_h; p.b_sl = b->stride_l;
  p.g = g; p.f = f; p.g_sb = g_sb; p.g_sh = g_sh; p.f_sb = f_sb; p.f_sh = f_sh;
  p.weight = weight; p.L = L; p.keep = keep; p.recent = recent;
  p.index = static_cast<int32_t*>(workspace); p.B = (int)B; p.H = (int)H; p.status = status;
  return launched(sisa::launch_paged_fill(p, static_cast<cudaStream_t>(stream)), what);
}

}  // extern "C"
