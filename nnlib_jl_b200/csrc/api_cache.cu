// The C ABI of what stands around attention in a decoder layer (include/nnlib_b200.h): norm and rotation of heads, the
// 8-bit key / value cache and attention over it.  Argument checks and defaults, as in api.cu.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "common.cuh"
#include "launchers.h"

namespace nb200 {
namespace {

constexpr int64_t kMost = 0x7fffffffLL;

bool dtype_ok(int dt) { return dt == NNLIB_B200_F16 || dt == NNLIB_B200_BF16 || dt == NNLIB_B200_F32; }
int esize(int dt) { return dt == NNLIB_B200_F32 ? 4 : 2; }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// the arrays of a call: the first `always` are looked up on every call, the rest under NNLIB_B200_CHECK_POINTERS
int check_arrays(const void* const* ptrs, int always, int n) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return NNLIB_B200_CUDA_ERROR;
  }
  const int m = check_all_pointers() ? n : always;
  for (int i = 0; i < m; ++i)
    if (!on_current_device(ptrs[i], dev)) return NNLIB_B200_INVALID_ARG;
  return NNLIB_B200_OK;
}

// strides in elements, 0 = dense; false: rows or batches would overlap
bool strides(int64_t width, int64_t L, int64_t sl, int64_t sb, long long* out_l, long long* out_b) {
  *out_l = sl ? sl : width;
  *out_b = sb ? sb : *out_l * L;
  return *out_l >= width && *out_b >= 0;
}

int resolve_norm_rope(const nnlib_b200_norm_rope_params* p, bool bwd, NormRopeArgs* out) {
  if (!p || p->struct_size != sizeof(*p)) return NNLIB_B200_INVALID_ARG;
  if (!dtype_ok(p->dtype) || (p->wdtype != p->dtype && p->wdtype != NNLIB_B200_F32)) return NNLIB_B200_INVALID_ARG;
  if (p->d < 2 || p->d % 2 || p->rot < 0 || p->rot % 2 || p->rot > p->d) return NNLIB_B200_INVALID_ARG;
  if (p->Hq < 0 || p->Hk < 0 || p->Hq + p->Hk < 1 || p->L < 0 || p->B < 0) return NNLIB_B200_INVALID_ARG;
  if (p->d > 256) return NNLIB_B200_UNSUPPORTED_SHAPE;
  if (p->Hq > kMost / p->d || p->Hk > kMost / p->d || p->L > kMost || p->B > kMost || (p->L && p->B > kMost / p->L / std::max<int64_t>(1, std::max(p->Hq, p->Hk))))
    return NNLIB_B200_INVALID_ARG;
  if (!(p->eps >= 0.f) || std::isinf(p->eps)) return NNLIB_B200_INVALID_ARG;
  if (p->start0 < -kMost || p->start0 > kMost) return NNLIB_B200_INVALID_ARG;
  NormRopeArgs a;
  std::memset(&a, 0, sizeof(a));
  a.d = (int)p->d; a.rot = (int)p->rot; a.L = (int)p->L;
  a.tokens = p->L * p->B;
  a.interleaved = p->interleaved ? 1 : 0;
  a.wdtype = p->wdtype;
  a.eps = p->eps;
  a.freqs = p->freqs;
  a.positions = p->positions;
  a.pos_sl = p->positions_stride[0];
  a.pos_sb = p->positions_stride[1];
  if (a.pos_sl < 0 || a.pos_sb < 0) return NNLIB_B200_INVALID_ARG;
  a.start = p->start;
  a.start0 = p->start0;
  NormRopeSide& q = a.side[0];
  NormRopeSide& k = a.side[1];
  q.heads = (int)p->Hq; k.heads = (int)p->Hk;
  q.x = p->q; k.x = p->k;
  q.dy = p->dyq; k.dy = p->dyk;
  q.out = bwd ? p->dq : p->yq; k.out = bwd ? p->dk : p->yk;
  q.g = p->gq; k.g = p->gk;
  q.dg = p->dgq; k.dg = p->dgk;
  if (!strides(p->Hq * p->d, p->L, p->q_stride_l, p->q_stride_b, &q.sl, &q.sb) ||
      !strides(p->Hk * p->d, p->L, p->k_stride_l, p->k_stride_b, &k.sl, &k.sb) ||
      !strides(p->Hq * p->d, p->L, p->dyq_stride_l, p->dyq_stride_b, &q.dsl, &q.dsb) ||
      !strides(p->Hk * p->d, p->L, p->dyk_stride_l, p->dyk_stride_b, &k.dsl, &k.dsb))
    return NNLIB_B200_INVALID_ARG;
  for (const NormRopeSide& s : a.side) {
    if (!s.heads) continue;
    if (bwd && !s.dg) return NNLIB_B200_INVALID_ARG;
    if (a.tokens && (!s.x || !s.out || !s.g || (bwd && !s.dy))) return NNLIB_B200_INVALID_ARG;
    const uintptr_t z = esize(p->dtype);
    if (!aligned(s.x, z) || !aligned(s.out, z) || !aligned(s.dy, z) || !aligned(s.g, esize(p->wdtype)) || !aligned(s.dg, esize(p->wdtype)))
      return NNLIB_B200_INVALID_ARG;
  }
  if (a.tokens && a.rot && !a.freqs) return NNLIB_B200_INVALID_ARG;
  if (!aligned(a.freqs, 8) || !aligned(a.positions, 4) || !aligned(a.start, 4)) return NNLIB_B200_INVALID_ARG;
  *out = a;
  return NNLIB_B200_OK;
}

int check_norm_rope_arrays(const NormRopeArgs& a) {
  const NormRopeSide& s = a.side[a.side[0].heads ? 0 : 1];
  const void* all[] = {s.x, s.out, a.side[0].heads ? a.side[0].x : nullptr, a.side[1].heads ? a.side[1].x : nullptr,
                       a.side[0].heads ? a.side[0].out : nullptr, a.side[1].heads ? a.side[1].out : nullptr,
                       a.side[0].dy, a.side[1].dy, a.side[0].g, a.side[1].g, a.side[0].dg, a.side[1].dg,
                       a.freqs, a.positions, a.start};
  return check_arrays(all, 2, 15);
}

int resolve_cache(const nnlib_b200_cache* c, CacheArgs* out) {
  if (!c || c->struct_size != sizeof(*c)) return NNLIB_B200_INVALID_ARG;
  if (c->code != NNLIB_B200_INT8 && c->code != NNLIB_B200_E4M3) return NNLIB_B200_INVALID_ARG;
  if (c->d < 1 || c->H < 1 || c->pages < 0 || c->B < 0 || c->rows < 0 || c->table_stride < 0) return NNLIB_B200_INVALID_ARG;
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1))) return NNLIB_B200_INVALID_ARG;
  if (c->d % 16 || c->d > 256) return NNLIB_B200_UNSUPPORTED_SHAPE;
  if (c->H > 32767 || c->B > 32767 || c->pages > kMost) return NNLIB_B200_INVALID_ARG;
  if (c->rows > (kMost - 4095) / c->page) return NNLIB_B200_INVALID_ARG;
  CacheArgs a;
  std::memset(&a, 0, sizeof(a));
  a.code = c->code;
  a.d = (int)c->d; a.H = (int)c->H; a.B = (int)c->B;
  a.row = c->d * c->H;
  a.pages = c->pages;
  while ((1 << a.log_page) < c->page) ++a.log_page;
  a.table = c->table;
  a.table_stride = c->table_stride ? c->table_stride : c->rows;
  a.rows = c->rows;
  a.run = c->B > 0 ? c->pages / c->B : 0;
  if (!c->table && c->B > 0 && c->rows > c->pages / c->B) return NNLIB_B200_INVALID_ARG;
  if (c->table && a.table_stride < c->rows && c->B > 1) return NNLIB_B200_INVALID_ARG;
  a.codes[0] = static_cast<unsigned char*>(c->k_codes);
  a.codes[1] = static_cast<unsigned char*>(c->v_codes);
  a.scale[0] = c->k_scale;
  a.scale[1] = c->v_scale;
  if (c->pages > 0 && (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale)) return NNLIB_B200_INVALID_ARG;
  if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) ||
      !aligned(c->table, 4))
    return NNLIB_B200_INVALID_ARG;
  *out = a;
  return NNLIB_B200_OK;
}

int resolve_tokens(const CacheArgs& c, const nnlib_b200_cache_tokens* p, CacheTokens* out) {
  if (!p || p->struct_size != sizeof(*p) || !dtype_ok(p->dtype)) return NNLIB_B200_INVALID_ARG;
  if (p->L < 0 || p->L > kMost - 4096 || p->start0 < -kMost || p->start0 > kMost) return NNLIB_B200_INVALID_ARG;
  CacheTokens t;
  std::memset(&t, 0, sizeof(t));
  t.x[0] = p->k;
  t.x[1] = p->v;
  if (!strides(c.row, p->L, p->k_stride_l, p->k_stride_b, &t.sl[0], &t.sb[0]) ||
      !strides(c.row, p->L, p->v_stride_l, p->v_stride_b, &t.sl[1], &t.sb[1]))
    return NNLIB_B200_INVALID_ARG;
  t.start = p->start;
  t.start0 = p->start0;
  t.count = p->count;
  t.lens = p->lens;
  t.L = (int)p->L;
  const uintptr_t z = esize(p->dtype);
  if (!aligned(p->k, z) || !aligned(p->v, z) || !aligned(p->start, 4) || !aligned(p->count, 4) || !aligned(p->lens, 4))
    return NNLIB_B200_INVALID_ARG;
  if (t.L > 0 && c.B > 0) {
    if (!p->k || !p->v) return NNLIB_B200_INVALID_ARG;
    const void* all[] = {p->k, c.codes[0], p->v, c.codes[1], c.scale[0], c.scale[1], c.table, p->start, p->count, p->lens};
    const int rc = check_arrays(all, 2, 10);
    if (rc) return rc;
  }
  *out = t;
  return NNLIB_B200_OK;
}

int resolve_attn(const CacheArgs& c, const nnlib_b200_cache_attn_params* p, bool launching, CacheAttnArgs* out) {
  if (!p || p->struct_size != sizeof(*p) || !dtype_ok(p->dtype)) return NNLIB_B200_INVALID_ARG;
  if (p->Hq < 1 || p->Hq % c.H || p->L < 0) return NNLIB_B200_INVALID_ARG;
  if (p->Hq > kMost / c.d || p->L > kMost / p->Hq || (c.B && p->L * p->Hq > kMost / c.B)) return NNLIB_B200_INVALID_ARG;
  if (!(p->scale >= 0.f) || std::isinf(p->scale)) return NNLIB_B200_INVALID_ARG;
  CacheAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.c = c;
  if (c.pages == 0) a.c.rows = 0;            // a pool without a page has no address to read in a page's place
  a.q = p->q;
  a.x = p->x;
  if (!strides(p->Hq * c.d, p->L, p->q_stride_l, p->q_stride_b, &a.q_sl, &a.q_sb) ||
      !strides(p->Hq * c.d, p->L, p->x_stride_l, p->x_stride_b, &a.x_sl, &a.x_sb))
    return NNLIB_B200_INVALID_ARG;
  a.lens = p->lens;
  a.len0 = p->len0;
  a.start = p->start;
  a.scale = p->scale == 0.f ? (float)(1.0 / std::sqrt((double)c.d)) : p->scale;
  a.causal = p->causal ? 1 : 0;
  a.nan_fm = p->nan_on_fully_masked ? 1 : 0;
  a.Hq = (int)p->Hq;
  a.L = (int)p->L;
  a.lse = p->lse;
  a.status = p->status;
  const uintptr_t z = esize(p->dtype);
  if (!aligned(p->q, z) || !aligned(p->x, z) || !aligned(p->lens, 4) || !aligned(p->start, 4) || !aligned(p->lse, 4) || !aligned(p->status, 4))
    return NNLIB_B200_INVALID_ARG;
  if (a.L > 0 && c.B > 0) {
    if (!p->q || !p->x) return NNLIB_B200_INVALID_ARG;
    if (launching) {
      const void* all[] = {p->q, p->x, c.codes[0], c.codes[1], c.scale[0], c.scale[1], c.table, p->lens, p->start, p->lse, p->status};
      const int rc = check_arrays(all, 2, 11);
      if (rc) return rc;
    }
  }
  *out = a;
  return NNLIB_B200_OK;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

int nnlib_b200_norm_rope(const nnlib_b200_norm_rope_params* p, void* stream) {
  NormRopeArgs a;
  int rc = resolve_norm_rope(p, false, &a);
  if (rc) return rc;
  if (a.tokens == 0) return NNLIB_B200_OK;
  rc = check_norm_rope_arrays(a);
  if (rc) return rc;
  return finish(norm_rope(a, p->dtype, false, (cudaStream_t)stream));
}

size_t nnlib_b200_norm_rope_bwd_workspace_bytes(const nnlib_b200_norm_rope_params* p) {
  NormRopeArgs a;
  if (resolve_norm_rope(p, true, &a) != NNLIB_B200_OK) return 0;
  return norm_rope_workspace_bytes(a, esize(p->dtype));
}

int nnlib_b200_norm_rope_bwd(const nnlib_b200_norm_rope_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  NormRopeArgs a;
  int rc = resolve_norm_rope(p, true, &a);
  if (rc) return rc;
  const size_t need = norm_rope_workspace_bytes(a, esize(p->dtype));
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return NNLIB_B200_WORKSPACE_TOO_SMALL;
  rc = check_norm_rope_arrays(a);
  if (rc) return rc;
  a.ws = static_cast<float*>(workspace);
  return finish(norm_rope(a, p->dtype, true, (cudaStream_t)stream));
}

int nnlib_b200_cache_write(const nnlib_b200_cache* c, const nnlib_b200_cache_tokens* t, void* stream) {
  CacheArgs a;
  CacheTokens k;
  int rc = resolve_cache(c, &a);
  if (!rc) rc = resolve_tokens(a, t, &k);
  if (rc) return rc;
  if (k.L == 0 || a.B == 0 || a.rows == 0) return NNLIB_B200_OK;
  return finish(cache_write(a, k, t->dtype, (cudaStream_t)stream));
}

int nnlib_b200_cache_read(const nnlib_b200_cache* c, const nnlib_b200_cache_tokens* t, void* stream) {
  CacheArgs a;
  CacheTokens k;
  int rc = resolve_cache(c, &a);
  if (!rc) rc = resolve_tokens(a, t, &k);
  if (rc) return rc;
  if (k.L == 0 || a.B == 0) return NNLIB_B200_OK;
  return finish(cache_read(a, k, t->dtype, (cudaStream_t)stream));
}

size_t nnlib_b200_cache_attn_workspace_bytes(const nnlib_b200_cache* c, const nnlib_b200_cache_attn_params* p) {
  CacheArgs k;
  CacheAttnArgs a;
  if (resolve_cache(c, &k) || resolve_attn(k, p, false, &a) || a.L == 0 || k.B == 0) return 0;
  return cache_attn_workspace_bytes(a, p->dtype);
}

int nnlib_b200_cache_attn_path(const nnlib_b200_cache* c, const nnlib_b200_cache_attn_params* p) {
  CacheArgs k;
  CacheAttnArgs a;
  int rc = resolve_cache(c, &k);
  if (!rc) rc = resolve_attn(k, p, false, &a);
  if (rc) return rc;
  return cache_attn_umma_path(a, p->dtype) ? NNLIB_B200_PATH_UMMA : NNLIB_B200_PATH_SIMT;
}

int nnlib_b200_cache_attn(const nnlib_b200_cache* c, const nnlib_b200_cache_attn_params* p, void* workspace,
                          size_t workspace_bytes, void* stream) {
  CacheArgs k;
  CacheAttnArgs a;
  int rc = resolve_cache(c, &k);
  if (!rc) rc = resolve_attn(k, p, true, &a);
  if (rc) return rc;
  if (a.L == 0 || k.B == 0) return NNLIB_B200_OK;
  const size_t need = cache_attn_workspace_bytes(a, p->dtype);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return NNLIB_B200_WORKSPACE_TOO_SMALL;
  a.ws = static_cast<float*>(workspace);
  if (log_calls())
    std::fprintf(stderr, "[nnlib_b200] cache_attn d=%d H=%d Hq=%d L=%d B=%d causal=%d -> %s\n", k.d, k.H, a.Hq, a.L, k.B, a.causal,
                 cache_attn_umma_path(a, p->dtype) ? "tcgen05" : "streamed keys");
  return finish(cache_attn(a, p->dtype, (cudaStream_t)stream));
}

}  // extern "C"
