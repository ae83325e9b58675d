// Host-side launch functions of every kernel family, shared between the
// translation units and the C ABI in api.cu.
#pragma once
#include <cuda_runtime.h>
#include "common.cuh"

namespace nb200 {

// argument check of the x + alpha composites (api.cu): everything attn_fwd and attn_scores would reject
int attention_validate(const nnlib_b200_attn_params* p, bool launching = true);
int attention_both(const nnlib_b200_attn_params* p, void* stream);

// CUDA-core kernels (attn_simt.cu)
bool simt_supports(int d, int dv);
cudaError_t simt_fwd(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t simt_stats(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t simt_scores(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t simt_apply(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t causal_fill(unsigned char* m, long long L, cudaStream_t st);
cudaError_t causal_check(const unsigned char* m, long long L, int* flag, cudaStream_t st);

// tiled CUDA-core kernels, head sizes up to 128 (attn_fma.cu, attn_bwd_fma.cu)
bool fma_supports(int d, int dv);
cudaError_t fma_fwd(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t fma_stats(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t fma_scores(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t fma_apply(const AttnArgs& a, int dtype, cudaStream_t st);
int fma_split_count(const AttnArgs& a, int dtype);       // blocks per unit of the split-key forward (1: not split)
size_t fma_split_workspace_bytes(const AttnArgs& a, int dtype);
cudaError_t fma_split(const AttnArgs& a, int dtype, cudaStream_t st);   // a.ws holds the workspace
bool fma_row_supports(const AttnArgs& a, int dtype);     // x, alpha and lse in one pass (short key sequences)
cudaError_t fma_row(const AttnArgs& a, int dtype, cudaStream_t st);
size_t fma_bwd_workspace_bytes(const AttnArgs& a);
int fma_bwd_chunk(const AttnArgs& a);                     // query tiles of a block of the one-pass form
// a.ws set: one pass, partial results in the workspace (Float32)
cudaError_t fma_bwd(const AttnArgs& a, const BwdArgs& g, int dtype, cudaStream_t st);

// backward on CUDA cores (attn_bwd_simt.cu)
bool simt_bwd_supports(int d, int dv);
cudaError_t simt_bwd(const AttnArgs& a, const BwdArgs& g, int dtype, cudaStream_t st);

// tcgen05 + TMA kernels (attn_umma.cu)
const char* umma_fwd_reject_reason(const AttnArgs& a, int dtype, bool need_v);
cudaError_t umma_fwd(const AttnArgs& a, int dtype, bool stats_only, cudaStream_t st);
cudaError_t umma_scores(const AttnArgs& a, int dtype, cudaStream_t st);
bool umma_apply_supports(const AttnArgs& a, int dtype);
cudaError_t umma_apply(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t umma_take_abort(int* out, cudaStream_t st);
cudaError_t umma_wait_runout(unsigned long long limit_ns, int* status, cudaStream_t st);

// tcgen05 + TMA kernels for other head sizes and for Float32 arrays on the TF32 path (attn_tile.cu)
const char* tile_reject_reason(const AttnArgs& a, int dtype, bool need_v, bool allow_tf32);
cudaError_t tile_fwd(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t tile_stats(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t tile_scores(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t tile_take_abort(int* out, cudaStream_t st);
int tile_split_count(const AttnArgs& a);                 // 0: the split-key forward does not apply (Lq > 128)
size_t tile_split_workspace_bytes(const AttnArgs& a);
cudaError_t tile_split(const AttnArgs& a, int dtype, cudaStream_t st);   // a.ws holds the workspace

// at most 16 queries, 16-bit arrays, no side input: keys streamed through warp-level products (attn_decode.cu)
bool decode_supports(const AttnArgs& a, int dtype);
int decode_split_count(const AttnArgs& a);
bool decode_leaves(const AttnArgs& a, long long units);  // better left to the two-tile forward, in a call of so many units
size_t decode_workspace_bytes(const AttnArgs& a);        // 0: too few keys to split
cudaError_t decode_fwd(const AttnArgs& a, int dtype, int n_splits, cudaStream_t st);   // a.ws holds the workspace

// x and alpha in one pass when a query's whole score row fits in tensor memory (attn_short.cu)
bool short_supports(const AttnArgs& a, int dtype);
cudaError_t short_attention(const AttnArgs& a, int dtype, cudaStream_t st);
cudaError_t short_take_abort(int* out, cudaStream_t st);

// tcgen05 backward kernels (attn_bwd_umma.cu)
bool umma_bwd_supports(const AttnArgs& a, const BwdArgs& g, int dtype);
cudaError_t umma_bwd(const AttnArgs& a, const BwdArgs& g, int dtype, cudaStream_t st);
cudaError_t umma_bwd_take_abort(int* out, cudaStream_t st);

// one-pass tcgen05 backward, same calls, with a workspace in a.ws (attn_bwd_fused.cu)
size_t umma_bwd_fused_workspace_bytes(const AttnArgs& a);
cudaError_t umma_bwd_fused(const AttnArgs& a, const BwdArgs& g, int dtype, cudaStream_t st);
cudaError_t umma_bwd_fused_take_abort(int* out, cudaStream_t st);

// strided-batched matrix product: tcgen05 kernel for 16-bit arrays (gemm_umma.cu), CUDA-core kernel for the rest
// (gemm_fma.cu)
const char* gemm_umma_reject_reason(const GemmArgs& g, int dtype);
cudaError_t gemm_umma(const GemmArgs& g, int dtype, cudaStream_t st);
cudaError_t gemm_simt(const GemmArgs& g, int dtype, cudaStream_t st);
bool gemm_mma_supports(const GemmArgs& g, int dtype);    // 16-bit, any alignment: warp-level products (gemm_mma.cu)
cudaError_t gemm_mma(const GemmArgs& g, int dtype, cudaStream_t st);
cudaError_t gemm_take_abort(int* out, cudaStream_t st);

// softmax / logsoftmax over one dimension (softmax.cu)
cudaError_t softmax_forward(int dtype, bool log, const void* x, void* y, long long inner, long long n, long long outer,
                            cudaStream_t st);
cudaError_t softmax_backward(int dtype, bool log, const void* dy, const void* y, void* dx, long long inner, long long n,
                             long long outer, cudaStream_t st);

// helpers of the C ABI (api.cu)
int finish(cudaError_t e);                                // a return code, remembering what failed
bool on_current_device(const void* ptr, int dev);         // NULL passes
bool check_all_pointers();
bool log_calls();
bool force_simt();

// norm and rotation of heads (norm_rope.cu); a side is the queries or the keys
struct NormRopeSide {
  const void* x;
  const void* dy;            // pullback: the cotangent
  void* out;                 // forward: the result, pullback: the gradient of x; dense
  const void* g;
  void* dg;
  long long sl, sb, dsl, dsb;
  int heads;
  int chunk;                 // filled in by the launcher: heads that a warp takes of a token
};
struct NormRopeArgs {
  NormRopeSide side[2];
  const double* freqs;
  const int* positions;
  long long pos_sl, pos_sb;
  const int* start;
  long long start0;
  long long tokens;          // L * B
  float* ws;                 // pullback: d floats for each block
  float eps;
  int d, rot, L, interleaved, wdtype;
  int lanes, blocks_q;       // filled in by the launcher
};
size_t norm_rope_workspace_bytes(NormRopeArgs a, int esize);
cudaError_t norm_rope(NormRopeArgs a, int dtype, bool bwd, cudaStream_t st);

// 8-bit cache (cache.cu): what nnlib_b200_cache says, checked
struct CacheArgs {
  unsigned char* codes[2];   // keys, values
  float* scale[2];
  const int* table;
  long long table_stride, pages, row;   // row: bytes of a token, d * H
  long long rows;            // pages of a sequence
  long long run;             // without a table: pages from one sequence's first to the next one's
  int code, d, H, B, log_page;
};
struct CacheTokens {
  void* x[2];
  long long sl[2], sb[2];
  const int* start;
  long long start0;
  const int* count;
  const int* lens;
  int L;
};
cudaError_t cache_write(const CacheArgs& c, const CacheTokens& t, int dtype, cudaStream_t st);
cudaError_t cache_read(const CacheArgs& c, const CacheTokens& t, int dtype, cudaStream_t st);

// attention over it
struct CacheAttnArgs {
  CacheArgs c;
  const void* q;
  void* x;
  long long q_sl, q_sb, x_sl, x_sb;
  const int* lens;
  const int* start;
  long long len0;
  float* lse;
  float* ws;
  int* status;
  float scale;
  int causal, nan_fm, Hq, L;
};
size_t cache_attn_workspace_bytes(const CacheAttnArgs& a, int dtype);   // (cache_attn.cu)
cudaError_t cache_attn(CacheAttnArgs a, int dtype, cudaStream_t st);          // a.ws holds the workspace
bool cache_attn_umma_path(const CacheAttnArgs& a, int dtype);                 // which of the two it takes
bool cache_umma_supports(const CacheAttnArgs& a, int dtype);                  // tcgen05 (cache_attn_umma.cu): 16-bit, d <= 128
int cache_umma_splits(const CacheAttnArgs& a);
bool cache_umma_parts(const CacheAttnArgs& a, int dtype, int splits);         // it needs a workspace
cudaError_t cache_umma(const CacheAttnArgs& a, int dtype, int splits, cudaStream_t st);   // partial results only, if splits > 1
cudaError_t cache_umma_take_abort(int* out, cudaStream_t st);

// ---- ragged groups of columns (api_experts.cu checks, route.cu and grouped_*.cu compute) ----
struct RouteArgs {
  const void* logits;
  long long stride;
  const float* bias;
  const unsigned char* mask;
  float* weights;
  int* experts;
  int* offsets;
  int* columns;
  int* position;
  const float* dweights;
  void* dlogits;
  int* ws;                   // counts (G, blocks), totals (G)
  int G, N, k, normalize;
  int blocks, per_block, vec, k_up;   // filled in by the launcher
};
size_t route_workspace_bytes(const RouteArgs& a);
cudaError_t route(RouteArgs a, int dtype, cudaStream_t st);
cudaError_t route_bwd(const RouteArgs& a, int dtype, cudaStream_t st);

struct CombineArgs {
  const void* Y;
  const int* position;
  const float* weights;
  void* y;
  const int* columns;
  const void* dy;
  void* dY;
  float* dweights;
  long long Y_stride, y_stride, dy_stride;
  int E, N, R, k;
};
cudaError_t combine(const CombineArgs& a, int dtype, cudaStream_t st);
cudaError_t combine_bwd(const CombineArgs& a, int dtype, cudaStream_t st);

// C[:, i] = scale * A[:, :, id(g)] X[:, columns[i]] for the columns i of run g, and, with `low`, what a low-rank pair adds
struct LowRank {
  const void* B;             // (M, r, n), or (r, M, n)
  long long ldb, strideB;
  const void* T;             // scale * A X: (r, N) Float32 (grouped_fma.cu), or as grouped_umma.cu lays it out
  long long ldt;
  const int* offsets;        // runs; NULL: of run_len columns each
  const int* ids;
  long long run_len;
  int transB, r, n, runs;
};
struct GroupedArgs {
  const void* A;
  const void* X;
  void* C;
  long long lda, strideA, ldx, ldc;
  const int* offsets;        // NULL: runs of run_len columns each
  const int* ids;            // matrix of each run, outside 0 .. mats - 1: none (zeros); NULL: its own number
  const int* columns;
  const float* scale;        // of each matrix; NULL: scale0
  long long run_len;
  float scale0;
  int transA, zero_rest;
  int M, K, G, N, R, mats;   // G: runs, N: columns of X, R: columns of C
  LowRank low;               // r = 0: none
  int* status;
};
// Gradient of the matrices: A[:, :, a] = sum over the columns i of the runs of matrix a of C[:, i] X[:, columns[i]]^T
struct GroupedGradArgs {
  void* A;
  const void* X;
  const void* C;
  long long lda, strideA, ldx, ldc;
  const int* offsets;
  const int* ids;
  const int* columns;
  long long run_len;
  int transA;
  int M, K, G, N, R, mats;
  int* status;
};
// CUDA cores (grouped_fma.cu): everything.  parts: Float32 (M, R, grouped_fma_splits(g)) instead of C, for join_parts
int grouped_fma_splits(const GroupedArgs& g);
cudaError_t grouped_fma(const GroupedArgs& g, int dtype, bool f32_out, float* parts, cudaStream_t st);
cudaError_t join_parts(const GroupedArgs& g, int dtype, int splits, const float* parts, const float* t, int t_splits, cudaStream_t st);   // (grouped_umma.cu)
cudaError_t grouped_fma_grad(const GroupedGradArgs& g, int dtype, bool f32_rows, bool f32_cols, cudaStream_t st);
// tcgen05 (grouped_umma.cu): 16-bit arrays
bool grouped_umma_supports(const GroupedArgs& g, int dtype);
size_t grouped_umma_workspace_bytes(const GroupedArgs& g);
cudaError_t grouped_umma(const GroupedArgs& g, int dtype, void* workspace, cudaStream_t st);
int low_width(int r, int dtype);                          // 16-bit elements of T for a column
size_t low_umma_bytes(const GroupedArgs& first, int dtype);   // T of all columns
size_t low_umma_workspace_bytes(const GroupedArgs& first);
// odd, look: where it is noted which matrices of the pairs of `look` have infinities or NaN
cudaError_t low_umma(const GroupedArgs& first, int dtype, void* T, void* workspace, bool behind, cudaStream_t st, unsigned char* odd = nullptr,
                     const GroupedArgs* look = nullptr);
size_t adapter_umma_workspace_bytes(const GroupedArgs& first, const GroupedArgs& main, bool keep);
cudaError_t adapter_umma(const GroupedArgs& first, GroupedArgs main, int dtype, bool keep, void* low, void* workspace, cudaStream_t st);
bool grouped_umma_grad_supports(const GroupedGradArgs& g, int dtype);
size_t grouped_umma_grad_workspace_bytes(const GroupedGradArgs& g, int fold);
// fold: C (1) or X (2) is T; behind: a kernel of this call is before it in the stream
cudaError_t grouped_umma_grad(const GroupedGradArgs& g, int dtype, int fold, void* workspace, bool behind, cudaStream_t st);
cudaError_t grouped_take_abort(int* out, cudaStream_t st);

}  // namespace nb200
