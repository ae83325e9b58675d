// The C ABI of products of ragged groups of columns (include/nnlib_b200.h): the router, its experts' products, their weighted
// sum, low-rank adapters.  Argument checks and defaults, as in api.cu.
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
bool extent(int64_t n) { return n >= 0 && n <= kMost; }
// the kernels' indexes are 32 bits wide and go up to a tile, or a block's share, beyond an extent
bool countable(int64_t n) { return n <= kMost - 65536; }

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

// `count` matrices of rows x cols, stored as they are or transposed
bool matrix_ok(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t stride, int64_t count, bool trans, int z) {
  if (rows == 0 || cols == 0 || count == 0) return true;
  return p && aligned(p, z) && ld >= (trans ? cols : rows) && stride >= 0 && ld < (1ll << 40) && stride < (1ll << 40);
}

// ------------------------------------------------------------------------------------------------- router
int resolve_route(const nnlib_b200_route_params* p, bool bwd, RouteArgs* out) {
  if (!p || p->struct_size != sizeof(*p) || !dtype_ok(p->dtype)) return NNLIB_B200_INVALID_ARG;
  if (p->G < 1 || p->N < 0 || p->k < 1 || p->k > p->G || p->logits_stride < 0) return NNLIB_B200_INVALID_ARG;
  if (p->G > 1024 || p->k > 32) return NNLIB_B200_UNSUPPORTED_SHAPE;
  if (p->N > kMost / p->k) return NNLIB_B200_INVALID_ARG;
  if (!countable(p->N * p->k)) return NNLIB_B200_UNSUPPORTED_SHAPE;
  RouteArgs a;
  std::memset(&a, 0, sizeof(a));
  a.logits = p->logits;
  a.stride = p->logits_stride ? p->logits_stride : p->G;
  if (a.stride < p->G) return NNLIB_B200_INVALID_ARG;
  a.bias = p->bias;
  a.mask = p->mask;
  a.weights = p->weights;
  a.experts = p->experts;
  a.offsets = p->offsets;
  a.columns = p->columns;
  a.position = p->position;
  a.dweights = p->dweights;
  a.dlogits = p->dlogits;
  a.G = (int)p->G; a.N = (int)p->N; a.k = (int)p->k;
  a.normalize = p->normalize ? 1 : 0;
  const int z = esize(p->dtype);
  if (!aligned(p->logits, z) || !aligned(p->bias, 4) || !aligned(p->weights, 4) || !aligned(p->experts, 4) || !aligned(p->offsets, 4) ||
      !aligned(p->columns, 4) || !aligned(p->position, 4) || !aligned(p->dweights, 4) || !aligned(p->dlogits, z))
    return NNLIB_B200_INVALID_ARG;
  if (a.N && (!p->logits || !p->weights || !p->experts)) return NNLIB_B200_INVALID_ARG;
  if (bwd) {
    if (a.N && (!p->dweights || !p->dlogits)) return NNLIB_B200_INVALID_ARG;
  } else if (!p->offsets || (a.N && (!p->columns || !p->position))) {
    return NNLIB_B200_INVALID_ARG;
  }
  *out = a;
  return NNLIB_B200_OK;
}

// ------------------------------------------------------------------------------------------------- grouped products
int resolve_grouped(const nnlib_b200_grouped_params* p, GroupedArgs* out) {
  if (!p || p->struct_size != sizeof(*p) || !dtype_ok(p->dtype)) return NNLIB_B200_INVALID_ARG;
  if (!extent(p->M) || !extent(p->K) || !extent(p->N) || !extent(p->R) || p->G < 0) return NNLIB_B200_INVALID_ARG;
  if (p->G > 32767 || !countable(p->M) || !countable(p->K) || !countable(p->N) || !countable(p->R)) return NNLIB_B200_UNSUPPORTED_SHAPE;
  const int z = esize(p->dtype);
  if (!matrix_ok(p->A, p->M, p->K, p->lda, p->strideA, p->G, p->transA != 0, z) || !matrix_ok(p->X, p->K, p->N, p->ldx, 0, 1, false, z) ||
      !matrix_ok(p->C, p->M, p->R, p->ldc, 0, 1, false, z))
    return NNLIB_B200_INVALID_ARG;
  if ((p->G > 0 && !p->offsets) || (!p->columns && p->R > p->N)) return NNLIB_B200_INVALID_ARG;
  if (!aligned(p->offsets, 4) || !aligned(p->columns, 4) || !aligned(p->status, 4)) return NNLIB_B200_INVALID_ARG;
  GroupedArgs a;
  std::memset(&a, 0, sizeof(a));
  a.A = p->A; a.X = p->X; a.C = p->C;
  a.lda = p->lda; a.strideA = p->strideA; a.ldx = p->ldx; a.ldc = p->ldc;
  a.offsets = p->offsets;
  a.columns = p->columns;
  a.scale0 = 1.f;
  a.transA = p->transA ? 1 : 0;
  a.zero_rest = p->zero_rest ? 1 : 0;
  a.M = (int)p->M; a.K = (int)p->K; a.G = (int)p->G; a.N = (int)p->N; a.R = (int)p->R;
  a.mats = a.G;
  a.status = p->status;
  *out = a;
  return NNLIB_B200_OK;
}
GroupedGradArgs grad_of(const GroupedArgs& a) {
  GroupedGradArgs g;
  std::memset(&g, 0, sizeof(g));
  g.A = const_cast<void*>(a.A); g.X = a.X; g.C = a.C;
  g.lda = a.lda; g.strideA = a.strideA; g.ldx = a.ldx; g.ldc = a.ldc;
  g.offsets = a.offsets; g.ids = a.ids; g.columns = a.columns; g.run_len = a.run_len;
  g.transA = a.transA;
  g.M = a.M; g.K = a.K; g.G = a.G; g.N = a.N; g.R = a.R; g.mats = a.mats;
  g.status = a.status;
  return g;
}
// Float16 / BFloat16 on the tensor cores, unless there are more runs than a block's table of them holds
bool on_umma(const GroupedArgs& a, int dtype) { return !force_simt() && grouped_umma_supports(a, dtype); }
bool on_umma(const GroupedGradArgs& a, int dtype) { return !force_simt() && grouped_umma_grad_supports(a, dtype); }
int workspace_ok(const void* ws, size_t bytes, size_t need) {
  return need && (!ws || bytes < need || !aligned(ws, 16)) ? NNLIB_B200_WORKSPACE_TOO_SMALL : NNLIB_B200_OK;
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
// On the CUDA cores, by way of Float32 parts of K where that pays (ws: fma_ws() bytes).  They are also the way for low-rank pairs that few columns
// share: the launch that adds the parts takes each column's pair by itself, a tile all of its columns' pairs one after the other (24 single
// columns, 304 x 160, rank 128: 20 us, 211 in the tile).  f32_out: C is Float32, whatever A and X are
int fma_parts(const GroupedArgs& a) {
  if (a.M == 0 || a.R == 0) return 0;
  const int splits = grouped_fma_splits(a);
  return splits > 1 || (a.low.r > 0 && a.R <= 512 && a.R <= 8ll * a.low.runs) ? splits : 0;
}
size_t fma_ws(const GroupedArgs& a) { return round256(sizeof(float) * fma_parts(a) * (size_t)a.R * a.M); }
cudaError_t fma_product(GroupedArgs a, int dtype, bool f32_out, void* ws, cudaStream_t st) {
  const int parts = fma_parts(a);
  if (parts == 0) return grouped_fma(a, dtype, f32_out, nullptr, st);
  const float* t = a.low.r > 0 ? static_cast<const float*>(a.low.T) : nullptr;
  GroupedArgs main = a;
  main.low.r = 0;
  const cudaError_t e = grouped_fma(main, dtype, f32_out, static_cast<float*>(ws), st);
  return e != cudaSuccess ? e : join_parts(a, f32_out ? NNLIB_B200_F32 : dtype, parts, static_cast<const float*>(ws), t, 1, st);
}

int check_grouped_arrays(const GroupedArgs& a) {
  const void* all[] = {a.C, a.X, a.A, a.offsets, a.columns, a.status};
  return check_arrays(all, 2, 6);
}

// ------------------------------------------------------------------------------------------------- combine
int resolve_combine(const nnlib_b200_combine_params* p, bool bwd, CombineArgs* out) {
  if (!p || p->struct_size != sizeof(*p) || !dtype_ok(p->dtype)) return NNLIB_B200_INVALID_ARG;
  if (p->E < 1 || !extent(p->E) || !extent(p->N) || !extent(p->R) || p->k < 1) return NNLIB_B200_INVALID_ARG;
  if (p->k > 32) return NNLIB_B200_UNSUPPORTED_SHAPE;
  if (p->N > kMost / p->k || p->R > kMost - 8) return NNLIB_B200_INVALID_ARG;
  if (!countable(p->E) || !countable(p->R)) return NNLIB_B200_UNSUPPORTED_SHAPE;
  CombineArgs a;
  std::memset(&a, 0, sizeof(a));
  a.Y = p->Y; a.y = p->y; a.dy = p->dy; a.dY = p->dY;
  a.position = p->position;
  a.weights = p->weights;
  a.columns = p->columns;
  a.dweights = p->dweights;
  a.Y_stride = p->Y_stride ? p->Y_stride : p->E;
  a.y_stride = p->y_stride ? p->y_stride : p->E;
  a.dy_stride = p->dy_stride ? p->dy_stride : p->E;
  a.E = (int)p->E; a.N = (int)p->N; a.R = (int)p->R; a.k = (int)p->k;
  const int z = esize(p->dtype);
  if (a.Y_stride < p->E || a.y_stride < p->E || a.dy_stride < p->E) return NNLIB_B200_INVALID_ARG;
  if (!aligned(p->Y, z) || !aligned(p->y, z) || !aligned(p->dy, z) || !aligned(p->dY, z) || !aligned(p->position, 4) ||
      !aligned(p->weights, 4) || !aligned(p->columns, 4) || !aligned(p->dweights, 4))
    return NNLIB_B200_INVALID_ARG;
  if (a.N && !p->position) return NNLIB_B200_INVALID_ARG;
  if (a.R && !p->Y && (!bwd || p->dweights)) return NNLIB_B200_INVALID_ARG;
  if (bwd) {
    if ((a.R && (!p->dY || !p->columns)) || (a.N && !p->dy)) return NNLIB_B200_INVALID_ARG;
  } else if (a.N && !p->y) {
    return NNLIB_B200_INVALID_ARG;
  }
  *out = a;
  return NNLIB_B200_OK;
}

// ------------------------------------------------------------------------------------------------- adapters
struct Adapters {
  GroupedArgs main;          // W X with the low-rank term; for the gradient of X W^T dC
  GroupedArgs first;         // the factor next to the columns: A X; for the gradient of X B^T dC
};

int resolve_adapter(const nnlib_b200_adapter_params* p, bool bwd, Adapters* out) {
  if (!p || p->struct_size != sizeof(*p) || !dtype_ok(p->dtype)) return NNLIB_B200_INVALID_ARG;
  if (!extent(p->M) || !extent(p->K) || !extent(p->N) || p->r < 1 || p->n < 0 || p->runs < 0 || p->run_len < 0) return NNLIB_B200_INVALID_ARG;
  if (p->r > 128 || p->n > 32767 || p->runs > (1 << 20) || !countable(p->M) || !countable(p->K) || !countable(p->N)) return NNLIB_B200_UNSUPPORTED_SHAPE;
  if (p->run_len > kMost) return NNLIB_B200_INVALID_ARG;
  const int z = esize(p->dtype);
  if (!matrix_ok(p->W, p->M, p->K, p->ldw, 0, 1, p->transW != 0, z) || !matrix_ok(p->A, p->r, p->K, p->lda, p->strideA, p->n, p->transA != 0, z) ||
      !matrix_ok(p->B, p->M, p->r, p->ldb, p->strideB, p->n, p->transB != 0, z))
    return NNLIB_B200_INVALID_ARG;
  if (p->runs > 0 && !p->ids) return NNLIB_B200_INVALID_ARG;
  if (!aligned(p->offsets, 4) || !aligned(p->ids, 4) || !aligned(p->scale, 4) || !aligned(p->status, 4)) return NNLIB_B200_INVALID_ARG;
  if (!bwd) {
    if (!matrix_ok(p->X, p->K, p->N, p->ldx, 0, 1, false, z) || !matrix_ok(p->C, p->M, p->N, p->ldc, 0, 1, false, z)) return NNLIB_B200_INVALID_ARG;
  } else {
    if (!matrix_ok(p->dC, p->M, p->N, p->lddc, 0, 1, false, z) || !matrix_ok(p->dX, p->K, p->N, p->K, 0, 1, false, z)) return NNLIB_B200_INVALID_ARG;
    if ((p->dA == nullptr) != (p->dB == nullptr) && p->M && p->K && p->n) return NNLIB_B200_INVALID_ARG;
    if (p->dA && !matrix_ok(p->X, p->K, p->N, p->ldx, 0, 1, false, z)) return NNLIB_B200_INVALID_ARG;
    if (!aligned(p->dA, z) || !aligned(p->dB, z)) return NNLIB_B200_INVALID_ARG;
  }
  Adapters a;
  std::memset(&a, 0, sizeof(a));
  GroupedArgs& m = a.main;
  GroupedArgs& f = a.first;
  f.offsets = p->offsets;
  f.ids = p->ids;
  f.run_len = p->run_len;
  f.scale = p->scale;
  f.scale0 = p->scale0;
  f.G = (int)p->runs; f.mats = (int)p->n;
  f.M = (int)p->r;
  f.N = f.R = m.N = m.R = (int)p->N;
  f.status = m.status = p->status;
  m.A = p->W; m.lda = p->ldw;
  m.G = m.mats = 1;
  m.run_len = p->N;
  m.scale0 = 1.f;
  LowRank& l = m.low;
  l.offsets = p->offsets;
  l.ids = p->ids;
  l.run_len = p->run_len;
  l.r = (int)p->r; l.n = (int)p->n; l.runs = (int)p->runs;
  if (!bwd) {
    m.M = (int)p->M; m.K = f.K = (int)p->K;
    m.transA = p->transW ? 1 : 0;
    m.X = f.X = p->X; m.ldx = f.ldx = p->ldx;
    m.C = p->C; m.ldc = p->ldc;
    f.A = p->A; f.lda = p->lda; f.strideA = p->strideA; f.transA = p->transA ? 1 : 0;
    l.B = p->B; l.ldb = p->ldb; l.strideB = p->strideB; l.transB = p->transB ? 1 : 0;
  } else {
    m.M = (int)p->K; m.K = f.K = (int)p->M;
    m.transA = p->transW ? 0 : 1;
    m.X = f.X = p->dC; m.ldx = f.ldx = p->lddc;
    m.C = p->dX; m.ldc = p->K;
    f.A = p->B; f.lda = p->ldb; f.strideA = p->strideB; f.transA = p->transB ? 0 : 1;
    l.B = p->A; l.ldb = p->lda; l.strideB = p->strideA; l.transB = p->transA ? 0 : 1;
  }
  *out = a;
  return NNLIB_B200_OK;
}
// on the tensor cores both products are, or neither: T is theirs
bool adapter_on_umma(const Adapters& a, int dtype) {
  GroupedArgs f = a.first;
  f.G = std::max(1, f.G);
  f.mats = std::max(1, f.mats);
  return on_umma(a.main, dtype) && on_umma(f, dtype);
}
bool has_pairs(const Adapters& a) { return a.first.G > 0 && a.first.mats > 0 && a.first.K > 0; }
size_t low_bytes(const Adapters& a, int dtype, bool umma) {
  return umma ? low_umma_bytes(a.first, dtype) : round256((size_t)a.first.R * 4 * (size_t)a.first.M);
}
// A X (or B^T dC) into `low`, then the product that adds B times it (A^T times it); `ws`: adapter_ws() bytes.  keep: `low` is read behind it.
cudaError_t adapter_products(Adapters& a, int dtype, bool umma, bool keep, void* low, void* ws, cudaStream_t st) {
  if (!has_pairs(a)) a.main.low.r = 0;
  if (umma) return adapter_umma(a.first, a.main, dtype, keep, low, ws, st);
  a.first.C = low;
  a.first.ldc = a.first.M;
  a.main.low.T = low;
  a.main.low.ldt = a.first.M;
  if (a.first.G > 0 && a.first.mats > 0) {             // (without features too: the gradients read it, as zeros)
    const cudaError_t e = fma_product(a.first, dtype, true, ws, st);
    if (e != cudaSuccess) return e;
  }
  return fma_product(a.main, dtype, false, ws, st);
}
size_t adapter_ws(Adapters& a, bool umma, bool keep) {
  if (!has_pairs(a)) a.main.low.r = 0;
  return umma ? adapter_umma_workspace_bytes(a.first, a.main, keep) : std::max(fma_ws(a.first), fma_ws(a.main));
}

// Gradients of the pairs: dA = (scale B^T dC) X^T, dB = dC (scale A X)^T.  `other`: A X for them.
struct PairGrads {
  GroupedArgs first;         // A X
  GroupedGradArgs a, b;
};
PairGrads pair_grads(const nnlib_b200_adapter_params* p, const Adapters& a, bool umma) {
  PairGrads o;
  o.first = a.first;
  o.first.A = p->A; o.first.lda = p->lda; o.first.strideA = p->strideA; o.first.transA = p->transA ? 1 : 0;
  o.first.K = (int)p->K;
  o.first.X = p->X; o.first.ldx = p->ldx;
  const long long wide = umma ? low_width((int)p->r, p->dtype) : p->r;
  o.a = grad_of(o.first);
  o.a.A = p->dA; o.a.lda = p->transA ? p->K : p->r; o.a.strideA = p->r * p->K;
  o.a.C = nullptr; o.a.ldc = wide;
  o.b = grad_of(o.first);
  o.b.A = p->dB; o.b.transA = p->transB ? 1 : 0; o.b.lda = p->transB ? p->r : p->M; o.b.strideA = p->M * p->r;
  o.b.M = (int)p->M; o.b.K = (int)p->r;
  o.b.C = p->dC; o.b.ldc = p->lddc;
  o.b.X = nullptr; o.b.ldx = wide;
  return o;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" {

size_t nnlib_b200_route_workspace_bytes(const nnlib_b200_route_params* p) {
  RouteArgs a;
  if (resolve_route(p, false, &a)) return 0;
  return route_workspace_bytes(a);
}
int nnlib_b200_route(const nnlib_b200_route_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  RouteArgs a;
  int rc = resolve_route(p, false, &a);
  if (rc) return rc;
  const size_t need = route_workspace_bytes(a);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return NNLIB_B200_WORKSPACE_TOO_SMALL;
  const void* all[] = {a.offsets, a.logits, a.bias, a.mask, a.weights, a.experts, a.columns, a.position};
  if ((rc = check_arrays(all, 2, 8))) return rc;
  a.ws = static_cast<int*>(workspace);
  return finish(route(a, p->dtype, (cudaStream_t)stream));
}
int nnlib_b200_route_bwd(const nnlib_b200_route_params* p, void* stream) {
  RouteArgs a;
  int rc = resolve_route(p, true, &a);
  if (rc || a.N == 0) return rc;
  const void* all[] = {a.dlogits, a.logits, a.weights, a.experts, a.dweights};
  if ((rc = check_arrays(all, 2, 5))) return rc;
  return finish(route_bwd(a, p->dtype, (cudaStream_t)stream));
}

size_t nnlib_b200_grouped_gemm_workspace_bytes(const nnlib_b200_grouped_params* p) {
  GroupedArgs a;
  if (resolve_grouped(p, &a)) return 0;
  return on_umma(a, p->dtype) ? grouped_umma_workspace_bytes(a) : fma_ws(a);
}
int nnlib_b200_grouped_gemm(const nnlib_b200_grouped_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  GroupedArgs a;
  int rc = resolve_grouped(p, &a);
  if (rc || a.M == 0 || a.R == 0) return rc;
  const bool umma = on_umma(a, p->dtype);
  if ((rc = workspace_ok(workspace, workspace_bytes, umma ? grouped_umma_workspace_bytes(a) : fma_ws(a)))) return rc;
  if ((rc = check_grouped_arrays(a))) return rc;
  if (log_calls())
    std::fprintf(stderr, "[nnlib_b200] grouped_gemm M=%d K=%d G=%d N=%d R=%d -> %s\n", a.M, a.K, a.G, a.N, a.R, umma ? "tcgen05" : "cuda-core");
  return finish(umma ? grouped_umma(a, p->dtype, workspace, (cudaStream_t)stream) : fma_product(a, p->dtype, false, workspace, (cudaStream_t)stream));
}
size_t nnlib_b200_grouped_gemm_grad_workspace_bytes(const nnlib_b200_grouped_params* p) {
  GroupedArgs a;
  if (resolve_grouped(p, &a)) return 0;
  const GroupedGradArgs g = grad_of(a);
  return on_umma(g, p->dtype) ? grouped_umma_grad_workspace_bytes(g, 0) : 0;
}
int nnlib_b200_grouped_gemm_grad(const nnlib_b200_grouped_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  GroupedArgs a;
  int rc = resolve_grouped(p, &a);
  if (rc || a.M == 0 || a.K == 0 || a.G == 0) return rc;
  if (a.G > 1 && a.strideA == 0) return NNLIB_B200_INVALID_ARG;        // (one matrix for all runs is read, not written)
  const GroupedGradArgs g = grad_of(a);
  const bool umma = on_umma(g, p->dtype);
  if (umma && (rc = workspace_ok(workspace, workspace_bytes, grouped_umma_grad_workspace_bytes(g, 0)))) return rc;
  if ((rc = check_grouped_arrays(a))) return rc;
  if (log_calls())
    std::fprintf(stderr, "[nnlib_b200] grouped_gemm_grad M=%d K=%d G=%d N=%d R=%d -> %s\n", a.M, a.K, a.G, a.N, a.R, umma ? "tcgen05" : "cuda-core");
  return finish(umma ? grouped_umma_grad(g, p->dtype, 0, workspace, false, (cudaStream_t)stream)
                     : grouped_fma_grad(g, p->dtype, false, false, (cudaStream_t)stream));
}

int nnlib_b200_combine(const nnlib_b200_combine_params* p, void* stream) {
  CombineArgs a;
  int rc = resolve_combine(p, false, &a);
  if (rc || a.N == 0) return rc;
  const void* all[] = {a.y, a.Y, a.position, a.weights};
  if ((rc = check_arrays(all, 2, 4))) return rc;
  return finish(combine(a, p->dtype, (cudaStream_t)stream));
}
int nnlib_b200_combine_bwd(const nnlib_b200_combine_params* p, void* stream) {
  CombineArgs a;
  int rc = resolve_combine(p, true, &a);
  if (rc || (a.N == 0 && a.R == 0)) return rc;
  const void* all[] = {a.dY, a.dy, a.Y, a.position, a.weights, a.columns, a.dweights};
  if ((rc = check_arrays(all, 2, 7))) return rc;
  return finish(combine_bwd(a, p->dtype, (cudaStream_t)stream));
}

size_t nnlib_b200_adapter_gemm_workspace_bytes(const nnlib_b200_adapter_params* p) {
  Adapters a;
  if (resolve_adapter(p, false, &a)) return 0;
  const bool umma = adapter_on_umma(a, p->dtype);
  return low_bytes(a, p->dtype, umma) + adapter_ws(a, umma, false);
}
int nnlib_b200_adapter_gemm(const nnlib_b200_adapter_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  Adapters a;
  int rc = resolve_adapter(p, false, &a);
  if (rc || a.main.M == 0 || a.main.N == 0) return rc;
  const bool umma = adapter_on_umma(a, p->dtype);
  const size_t low = low_bytes(a, p->dtype, umma);
  if ((rc = workspace_ok(workspace, workspace_bytes, low + adapter_ws(a, umma, false)))) return rc;
  const void* all[] = {p->C, p->X, p->W, p->A, p->B, p->offsets, p->ids, p->scale, p->status};
  if ((rc = check_arrays(all, 2, 9))) return rc;
  if (log_calls())
    std::fprintf(stderr, "[nnlib_b200] adapter_gemm M=%d K=%d N=%d r=%d runs=%d -> %s\n", a.main.M, a.main.K, a.main.N, a.first.M, a.first.G,
                 umma ? "tcgen05" : "cuda-core");
  return finish(adapter_products(a, p->dtype, umma, false, workspace, static_cast<char*>(workspace) + low, (cudaStream_t)stream));
}
size_t nnlib_b200_adapter_bwd_workspace_bytes(const nnlib_b200_adapter_params* p) {
  Adapters a;
  if (resolve_adapter(p, true, &a)) return 0;
  const bool umma = adapter_on_umma(a, p->dtype);
  size_t rest = adapter_ws(a, umma, true);
  const bool pairs = p->dA || p->dB;                       // (of no elements: NULL)
  if (!umma && pairs) rest = std::max(rest, fma_ws(pair_grads(p, a, false).first));
  if (umma && pairs) {
    const PairGrads g = pair_grads(p, a, true);
    rest = std::max({rest, low_umma_workspace_bytes(g.first), grouped_umma_grad_workspace_bytes(g.a, 1), grouped_umma_grad_workspace_bytes(g.b, 2)});
  }
  return 2 * low_bytes(a, p->dtype, umma) + rest;
}
int nnlib_b200_adapter_bwd(const nnlib_b200_adapter_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  Adapters a;
  int rc = resolve_adapter(p, true, &a);
  if (rc) return rc;
  const bool umma = adapter_on_umma(a, p->dtype);
  const size_t low = low_bytes(a, p->dtype, umma);
  if ((rc = workspace_ok(workspace, workspace_bytes, nnlib_b200_adapter_bwd_workspace_bytes(p)))) return rc;
  const void* all[] = {p->dX, p->dC, p->X, p->W, p->A, p->B, p->offsets, p->ids, p->scale, p->status, p->dA, p->dB};
  if ((rc = check_arrays(all, 2, 12))) return rc;
  if (log_calls())
    std::fprintf(stderr, "[nnlib_b200] adapter_bwd M=%lld K=%lld N=%lld r=%lld runs=%lld -> %s\n", (long long)p->M, (long long)p->K, (long long)p->N,
                 (long long)p->r, (long long)p->runs, umma ? "tcgen05" : "cuda-core");
  cudaStream_t st = (cudaStream_t)stream;
  char* of_dC = static_cast<char*>(workspace);             // scale * B^T dC
  char* of_X = of_dC + low;                                // scale * A X
  char* ws = of_X + low;
  if ((rc = finish(adapter_products(a, p->dtype, umma, true, of_dC, ws, st)))) return rc;
  if ((!p->dA && !p->dB) || a.first.mats == 0) return NNLIB_B200_OK;
  PairGrads g = pair_grads(p, a, umma);
  g.first.C = of_X;
  g.a.C = of_dC;
  g.b.X = of_X;
  if (!umma) {
    if ((rc = finish(fma_product(g.first, p->dtype, true, ws, st)))) return rc;
    if ((rc = finish(grouped_fma_grad(g.a, p->dtype, true, false, st)))) return rc;
    return finish(grouped_fma_grad(g.b, p->dtype, false, true, st));
  }
  if (has_pairs(a) && (rc = finish(low_umma(g.first, p->dtype, of_X, ws, true, st)))) return rc;
  if ((rc = finish(grouped_umma_grad(g.a, p->dtype, 1, ws, true, st)))) return rc;
  return finish(grouped_umma_grad(g.b, p->dtype, 2, ws, true, st));
}

}  // extern "C"
