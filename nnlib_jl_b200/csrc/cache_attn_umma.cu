// Attention over the 8-bit cache on the tensor cores: many queries at a time (parts of prompts, prompts).
//
// The arithmetic is that of cache_attn.cu: products of codes, which Float16 holds exactly, with the page's key scale on the
// logits and its value scale in the exponent.  Here the products are tcgen05.mma: a block owns 256 rows (two tiles of 128) of
// one sequence and cache head, row = query * G + head of the group, so that query heads that share keys share their tiles,
// and walks over the keys in tiles of 128:
//
//   warp 0       pages and scales of the next tiles, into shared memory
//   warp 1       issues every tcgen05.mma:  S_t = Q_t K_j^T (smem x smem -> TMEM),  O_t += W_t V_j (TMEM x smem -> TMEM)
//   warp 2       allocates / frees the 512 TMEM columns
//   warps 4-11   softmax of the two tiles (a thread owns a row), before that Q: rounded to Float16 after a power of two of
//                the row's own, after that x
//   warps 12-15  codes to Float16: K by two warps, V by two, from global memory through registers into the 128-byte
//                swizzled tiles the products read; both operands have a key's features in a row, so the code is the same
//
// Bound by the chain of a tile, its scores through the softmax and back into the products: 2.46 us a round of 128 keys (1024
// queries over 131072 tokens, 128 blocks of 1020 rounds) for 2048 cycles, 1.07 us, of tensor work.  A conversion is five
// instructions for four codes (Int8), 32768 codes a round, which is why it has warps of its own: the loads of a warp's next
// keys are under way while it converts some.  The copy engine could bring codes only, which would cost another pass through
// shared memory.  The length of the code counts: with the conversion of keys and of values written out each for itself every
// warp waited for instructions (2.30 ms, and 2.07 to 2.37 for changes that did no more work).  4096 queries over 8192 tokens of
// 4 sequences, 32 / 8 heads of 128, bf16 over Int8: 2.01 ms, 822 TFLOP/s; call after call for seconds 2.14 ms, at the power
// limit (994 W, 1.83 to 1.92 GHz).  (At 2.30 ms: sixteen softmax warps, two threads to a row, 2.26, but 512 queries over up to
// 16384 tokens in E4M3 0.75 instead of 0.64; eight converting warps 2.50 and 0.75.)
// A scale serves 16 keys at least (64 where the pages allow: SG), so a thread scales and sums by groups of SG keys.
// The products' additions cut off instead of rounding, always towards zero: behind n keys that one accumulator has summed x is
// short by some n 2^-27.2 where all values have one sign (1024 queries, values 0.5 and above: 2.1e-4 behind 32768 keys, 8.7e-4
// behind 131072; half a step of Float16 is 4.9e-4).  So every 32768 keys (BFloat16, whose step is eight times as large: 262144)
// the tensor memory's sums are added, rounded, to a Float32 row of the block's own in the workspace and begun anew, which
// keeps that below half of half a step for histories of any length.
// Weights leave with a factor of 2^10 and the running maximum is raised when it grew by more than 2^4: they are below 2^14
// and keep 11 bits down to 2^-24 of the largest.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "cache_codes.cuh"
#include "split_reduce.cuh"
#include "umma_shared.cuh"

namespace nb200 {

__device__ int g_cache_attn_abort = 0;   // sticky: a bounded wait ran out somewhere

namespace {

constexpr int kThreadsC = 512, kTiles = 2;
constexpr float kGap = 4.f, kBits = 10.f;
constexpr float kValueFloorU = 7.8886090522101181e-31f;   // 2^-100
constexpr int kMetaTiles = 8;
template <typename T>
constexpr int kFoldTiles = std::is_same<T, __half>::value ? 256 : 2048;      // tiles of keys that tensor memory sums up (a power of two)
constexpr int kWaves = 6;                // fewer waves of blocks than these are put in order by their lengths

struct __align__(16) PageMeta {
  float ks, lvs, ivs;     // key scale; log2(value scale) + kBits; 1 / value scale
  int page;               // -1: no tokens here
};

template <int D>
struct CfgC {
  static constexpr int kChunks = D / 64;
  static constexpr int kTileBytes = kChunks * kChunkBytes;
  static constexpr int kStagesK = D == 128 ? 2 : 4, kStagesV = D == 128 ? 3 : 4;
  static constexpr int kKOff = kTiles * kTileBytes, kVOff = kKOff + kStagesK * kTileBytes;
  static constexpr int kMetaOff = kVOff + kStagesV * kTileBytes;
  static constexpr int kBarOff = kMetaOff + kMetaTiles * 8 * (int)sizeof(PageMeta);
  static constexpr int kSmemBytes = kBarOff + 256 + 1024;
};
static_assert(CfgC<128>::kSmemBytes <= 232448, "shared memory budget");

struct BarsC {
  uint64_t q_full[kTiles], s_full[kTiles], p_half[kTiles][2], o_full[kTiles];
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t meta_full[2], meta_free[2];     // four tiles each
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(BarsC) <= 256, "barrier block");

template <int CODE>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& p0, uint32_t& p1) {
  if (CODE == NNLIB_B200_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(p0) : "r"(__byte_perm(u, 0x64646464u, 0x4140u)), "r"(0x64806480u));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(p1) : "r"(__byte_perm(u, 0x64646464u, 0x4342u)), "r"(0x64806480u));
  } else {
    asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %2; cvt.rn.f16x2.e4m3x2 %0, lo; cvt.rn.f16x2.e4m3x2 %1, hi; }"
        : "=r"(p0), "=r"(p1) : "r"(w));
  }
}

// One side's tiles: keys 128 (j_lo + j) .. of sequence b, head h, into the ring at `ring`.  Two warps, each one chunk of 64
// features (D = 128) or one half of the keys (D = 64); lane = (key of eight, piece of 16 features of four), which puts the
// stores of eight lanes, two neighbouring keys, on all banks.
// Keys that are not there, behind the last one or on pages that the pool does not have, read zeros (a NaN among E4M3's codes
// would spoil rows that give them no weight) or, behind the last one of a group of SG keys, that one once more.
__device__ const uint4 g_zero_codes[16] = {};

template <int D, int CODE, int SG>
__device__ __forceinline__ void convert_tiles(const CacheArgs& cc, const unsigned char* base, uint8_t* ring, const PageMeta* meta,
                                              uint64_t* full, uint64_t* empty, uint64_t* meta_full, volatile int* abort_flag,
                                              int stages, int w, int lane, int j_lo, int n_kv, int len) {
  constexpr int N = D == 128 ? 16 : 8, AHEAD = 8;     // loads of a tile, and how many are under way
  constexpr int kTileBytes = CfgC<D>::kTileBytes;
  const int key8 = lane >> 2, piece = lane & 3;
  const int feat = (D == 128 ? w * 64 : 0) + piece * 16;
  const int n0 = D == 128 ? 0 : w * 8;
  const bool feat_ok = feat < cc.d;
  uint8_t* out = ring + (D == 128 ? w * kChunkBytes : 0) + n0 * 1024 + key8 * 128;
  const int u0 = ((2 * piece) ^ key8) << 4, u1 = ((2 * piece + 1) ^ key8) << 4;
  const int T1 = (1 << cc.log_page) - 1;
  base += feat;
  uint4 raw[AHEAD];
  // 64 keys from number 64 hh of tile j on: where a group of SG of them begins, and its distance from key to key
  const unsigned char* group;
  int row, most;
  auto load = [&](uint4& r, int j, int hh, int i) {
    if (i % (SG / 8) == 0) {
      const int key = (j_lo + j) * kBN + hh * 64 + i * 8;
      const int page = meta[(j & (kMetaTiles - 1)) * 8 + hh * 4 + i / 2].page;
      const bool in = feat_ok && page >= 0;
      group = in ? base + (((long long)page << cc.log_page) + (key & T1)) * cc.row : reinterpret_cast<const unsigned char*>(g_zero_codes);
      row = in ? (int)cc.row : 0;
      most = len - 1 - key;
    }
    // (what little of L1 shared memory leaves is for the stack)
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
        : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(group + (long long)min((i % (SG / 8)) * 8 + key8, most) * row));
  };
  bool ok = n_kv > 0 && mbar_wait_warp(&meta_full[0], 0, abort_flag);
  if (ok) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(raw[i], 0, n0 / 8, i);
  }
  int s = 0;
  uint32_t phase = 1;                        // of the stage's last release: none is waited for in the first round
#pragma unroll 1
  for (int j = 0; j < n_kv && ok; ++j) {
    if (j >= stages) ok = mbar_wait_warp(&empty[s], phase, abort_flag);
    if (ok && j + 1 < n_kv && ((j + 1) & 3) == 0) ok = mbar_wait_warp(&meta_full[((j + 1) >> 2) & 1], ((j + 1) >> 3) & 1, abort_flag);
    if (!ok) break;
#pragma unroll 1
    for (int h = 0; h < N / AHEAD; ++h) {
      const bool last = h + 1 == N / AHEAD;
      const int jn = last ? j + 1 : j, hn = last ? n0 / 8 : n0 / 8 + h + 1;      // what is fetched meanwhile
      uint8_t* p = out + s * kTileBytes + h * (AHEAD * 1024);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const uint4 r = raw[i];
        uint4 a, b;
        codes4<CODE>(r.x, a.x, a.y);
        codes4<CODE>(r.y, a.z, a.w);
        codes4<CODE>(r.z, b.x, b.y);
        codes4<CODE>(r.w, b.z, b.w);
        if (jn < n_kv) load(raw[i], jn, hn, i);
        *reinterpret_cast<uint4*>(p + i * 1024 + u0) = a;
        *reinterpret_cast<uint4*>(p + i * 1024 + u1) = b;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&full[s]);
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  }
}

// SG: keys that certainly share a scale
template <typename T, int D, int CODE, int SG>
__global__ void __launch_bounds__(kThreadsC, 1) cache_attn_umma_kernel(const CacheAttnArgs a, const int splits, const int vec) {
  using C = CfgC<D>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kFold = kFoldTiles<T>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  BarsC* bars = reinterpret_cast<BarsC*>(smem + C::kBarOff);
  PageMeta* meta = reinterpret_cast<PageMeta*>(smem + C::kMetaOff);
  volatile int* abort_flag = &bars->abort_flag;
  const CacheArgs& cc = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.Hq / cc.H, rows = a.L * G, blocks = (rows + kTiles * kBM - 1) / (kTiles * kBM);
  // Heads of a sequence side by side; of their blocks the longest ones first.  Where there are a few waves of blocks only, and
  // not too many kinds of them, the order is that of the tiles of keys that they walk over, which the lengths on the device
  // say (512 queries over 16384, 14336, 12288 and 10240 tokens of 4 sequences, 256 blocks: pages in a run 643 us instead of 680,
  // through a table, E4M3 565 instead of 640); else the last
  // rows of all sequences come first.
  int item = blockIdx.x;
  const int h = item % cc.H;
  item /= cc.H;
  const int split = item % splits;
  item /= splits;
  int b = item % cc.B, block = blocks - 1 - item / cc.B;
  const long long cap = cc.rows << cc.log_page;
  auto length = [&](int b_) {
    const long long n = a.lens ? (long long)a.lens[b_] : a.len0;
    return (int)(n < 0 ? 0 : (n < cap ? n : cap));
  };
  const int kinds = blocks * cc.B;
  if (a.lens && kinds <= kThreadsC && gridDim.x <= kWaves * 148) {
    int* tiles = reinterpret_cast<int*>(smem);           // (where Q will be)
    int mine = 0;
    if ((int)threadIdx.x < kinds) {
      const int b_ = threadIdx.x % cc.B, last = min((blocks - (int)threadIdx.x / cc.B) * (kTiles * kBM), rows) - 1, n = length(b_);
      long long e = n;
      if (a.causal) e = min(e, (a.start ? (long long)a.start[b_] : (long long)n - a.L) + last / G + 1);
      mine = e <= 0 ? 0 : (int)((e + kBN - 1) / kBN);
      tiles[threadIdx.x] = mine;
    }
    __syncthreads();
    if ((int)threadIdx.x < kinds) {
      int rank = 0;
      for (int i = 0; i < kinds; ++i) rank += tiles[i] > mine || (tiles[i] == mine && i < (int)threadIdx.x);
      if (rank == item) bars->tmem_base = threadIdx.x;
    }
    __syncthreads();
    const int chosen = (int)bars->tmem_base;
    b = chosen % cc.B;
    block = blocks - 1 - chosen / cc.B;
    __syncthreads();                                     // before the tensor memory's address takes its place
  }
  const int row0 = block * (kTiles * kBM);

  const int len = length(b);
  const long long start = a.start ? (long long)a.start[b] : (long long)len - a.L;
  auto last_key = [&](int row) {      // the last key that a row sees, -1: none
    if (row >= rows) return -1;
    if (!a.causal) return len - 1;
    const long long e = start + row / G;
    return e < 0 ? -1 : (e < len ? (int)e : len - 1);
  };
  // this block's key tiles, and where each of its row tiles stops
  // (named, not an array: an index that is not a constant would put it into local memory)
  const int end0 = (last_key(min(row0 + kBM, rows) - 1) + kBN) / kBN;
  const int end1 = row0 + kBM < rows ? (last_key(min(row0 + 2 * kBM, rows) - 1) + kBN) / kBN : 0;
  const int share = (max(end0, end1) + splits - 1) / splits, j_lo = split * share;
  const int n_t0 = max(0, min(end0, j_lo + share) - j_lo), n_t1 = max(0, min(end1, j_lo + share) - j_lo);
  const int n_kv = max(n_t0, n_t1);

  if (threadIdx.x == 0) {
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&bars->q_full[t], 4);
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->p_half[t][0], 4);
      mbar_init(&bars->p_half[t][1], 4);
      mbar_init(&bars->o_full[t], 1);
      mbar_init(&bars->meta_full[t], 1);
      mbar_init(&bars->meta_free[t], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bars->k_full[s], 2);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 2);
      mbar_init(&bars->v_empty[s], 1);
    }
    bars->abort_flag = *reinterpret_cast<volatile int*>(&g_cache_attn_abort);
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const bool start_ok = (*abort_flag == 0);

  // registers: 128 x 64 + 256 x 168 + 128 x 112 = the 512 x 128 launched
  if (warp < 4) {
    setmaxnreg_dec<64>();
    if (start_ok && warp == 0) {
      // ---------------------------------------------------- pages and scales, four tiles at a time
      bool ok = true;
      for (int q = 0; 4 * q < n_kv && ok; ++q) {
        if (q >= 2) ok = mbar_wait_warp(&bars->meta_free[q & 1], ((q >> 1) - 1) & 1, abort_flag);
        if (!ok) break;
        const int j = 4 * q + (lane >> 3);
        const long long key = (long long)(j_lo + j) * kBN + (lane & 7) * 16;
        PageMeta m = {1.f, 0.f, 0.f, -1};
        if (key < len) {
          const long long page = cache_page(cc, b, key >> cc.log_page);
          float ks = __int_as_float(0x7fc00000), vs = ks;
          if (page >= 0) {
            ks = cc.scale[0][page * cc.H + h];
            vs = cc.scale[1][page * cc.H + h];
          }
          const float vse = vs >= kValueFloorU ? vs : (vs >= 0.f ? kValueFloorU : __int_as_float(0x7fc00000));
          m.ks = ks >= 0.f ? ks : __int_as_float(0x7fc00000);
          m.lvs = log2f(vse) + kBits;
          m.ivs = __fdiv_rn(1.f, vse);
          m.page = (int)page;
        }
        meta[(j & (kMetaTiles - 1)) * 8 + (lane & 7)] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->meta_full[q & 1]);
      }
    } else if (start_ok && warp == 1 && lane == 0 && n_kv > 0) {
      // ---------------------------------------------------- MMA issuer (descriptors as in attn_umma.cu)
      constexpr uint32_t idesc_qk = make_idesc_f16(false, kBM, kBN, false, false);
      constexpr uint32_t idesc_pv = make_idesc_f16(false, kBM, D, false, true);
      constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
      constexpr uint32_t lbo_k = (16u >> 4) << 16, lbo_v = (static_cast<uint32_t>(kChunkBytes) >> 4) << 16;
      constexpr uint32_t tile16 = C::kTileBytes >> 4;
      const uint32_t q_lo = (smem_u32(smem) >> 4) | lbo_k;
      const uint32_t k_lo = (smem_u32(smem + C::kKOff) >> 4) | lbo_k;
      const uint32_t v_lo = (smem_u32(smem + C::kVOff) >> 4) | lbo_v;
      // (the bases are made opaque, or the compiler keeps every descriptor of the loop in a register and spills them:
      // this thread's local loads then take longer than the products)
      auto issue_qk = [&](int t, int stage) {
        uint32_t ql = q_lo + t * tile16, kl = k_lo + stage * tile16, ts = tmem + t * kBN;
        asm volatile("" : "+r"(ql), "+r"(kl), "+r"(ts));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kChunkBytes >> 4) + (kk & 3) * 2;
          umma_ss_lohi(ts, ql + off, kl + off, desc_hi, idesc_qk, kk > 0 ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int t, int stage, int half, bool first) {
        uint32_t to = tmem + kTiles * kBN + t * D, tw = tmem + t * kBN + half * (kBN / 4), vl = v_lo + stage * tile16 + half * ((kBN / 32) * (2048 >> 4));
        asm volatile("" : "+r"(to), "+r"(tw), "+r"(vl));
#pragma unroll
        for (int kk = 0; kk < kBN / 32; ++kk)
          umma_ts_lohi(to, tw + kk * 8, vl + kk * (2048 >> 4), desc_hi, idesc_pv, (first && half == 0 && kk == 0) ? 0u : 1u);
      };
      bool ok = true;
      if (n_t0 > 0) ok = mbar_wait(&bars->q_full[0], 0, abort_flag);
      if (ok && n_t1 > 0) ok = mbar_wait(&bars->q_full[1], 0, abort_flag);
      if (ok) ok = mbar_wait(&bars->k_full[0], 0, abort_flag);
      if (ok) {
        tc_fence_after();
        if (n_t0 > 0) {
          issue_qk(0, 0);
          umma_commit(&bars->s_full[0]);
        }
        if (n_t1 > 0) {
          issue_qk(1, 0);
          umma_commit(&bars->s_full[1]);
        }
        umma_commit(&bars->k_empty[0]);
      }
#pragma unroll 1
      for (int j = 0; j < n_kv && ok; ++j) {
        BarsC* bb = bars;
        asm volatile("" : "+l"(bb));         // (nor every barrier's address)
        const int sv = j % C::kStagesV, sk = (j + 1) % C::kStagesK;
        const uint32_t par = j & 1;
        ok = mbar_wait(&bb->v_full[sv], (j / C::kStagesV) & 1, abort_flag);
        if (ok && j + 1 < n_kv) ok = mbar_wait(&bb->k_full[sk], ((j + 1) / C::kStagesK) & 1, abort_flag);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int nt = t == 0 ? n_t0 : n_t1;
          if (!ok || j >= nt) continue;
          ok = mbar_wait(&bb->p_half[t][0], par, abort_flag);
          if (!ok) continue;
          tc_fence_after();
          issue_pv(t, sv, 0, (j & (kFold - 1)) == 0);
          ok = mbar_wait(&bb->p_half[t][1], par, abort_flag);
          if (!ok) continue;
          tc_fence_after();
          issue_pv(t, sv, 1, false);
          if (j + 1 < nt) {
            issue_qk(t, sk);
            umma_commit(&bb->s_full[t]);
          } else {
            umma_commit(&bb->o_full[t]);
          }
        }
        if (!ok) break;
        umma_commit(&bb->v_empty[sv]);
        if (j + 1 < n_kv) umma_commit(&bb->k_empty[sk]);
        // everything of tiles up to j is done with: the pages and scales of j - 3 .. j may go
        if ((j & 3) == 3) umma_commit(&bb->meta_free[(j >> 2) & 1]);
      }
    }
  } else if (warp >= 12) {
    setmaxnreg_dec<112>();
    if (start_ok) {
      // (one piece of code for both sides: two keep every warp waiting for instructions)
      const bool v = warp >= 14;
      convert_tiles<D, CODE, SG>(cc, (v ? cc.codes[1] : cc.codes[0]) + (long long)h * cc.d, smem + (v ? C::kVOff : C::kKOff), meta,
                                 v ? bars->v_full : bars->k_full, v ? bars->v_empty : bars->k_empty, bars->meta_full, abort_flag,
                                 v ? C::kStagesV : C::kStagesK, (warp - 12) & 1, lane, j_lo, n_kv, len);
    }
  } else {
    setmaxnreg_inc<168>();
    const int t = (warp - 4) >> 2, nt = t == 0 ? n_t0 : n_t1;
    const int wq = warp & 3;
    if (start_ok && row0 + t * kBM < rows) {
      const uint32_t lane_base = tmem + (static_cast<uint32_t>(wq * 32) << 16);
      const uint32_t tS = lane_base + t * kBN, tO = lane_base + kTiles * kBN + t * D;
      // (rows behind the last one go along with it: looking nowhere they would take the slow way, at the edge, in every tile;
      // a warp of such rows alone only says that it has no weights to write)
      const int lim = last_key(min(row0 + t * kBM + wq * 32 + lane, rows - 1));
      const bool idle = row0 + t * kBM + wq * 32 >= rows;
      float crow = 0.f;
      if (nt > 0) {
        const int r = wq * 32 + lane, row = row0 + t * kBM + r;
        const bool row_ok = row < rows;
        const int i = row_ok ? row / G : 0, hq = h * G + (row_ok ? row % G : 0);
        // ------------------------------------------------ this row of Q, by a power of two to a largest element in [2^13, 2^14)
        const T* qp = reinterpret_cast<const T*>(a.q) + (long long)i * a.q_sl + (long long)b * a.q_sb + (long long)hq * cc.d;
        auto load8 = [&](int f, float (&v)[8]) {
          T e[8];
          if (vec) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(qp + f));
            memcpy(e, &raw, 16);
          } else {
#pragma unroll
            for (int u = 0; u < 8; ++u) e[u] = qp[f + u];
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = Elem<T>::to_f(e[u]);
        };
        float top = 0.f;
#pragma unroll
        for (int f = 0; f < D; f += 8)
          if (row_ok && f < cc.d) {
            float v[8];
            load8(f, v);
#pragma unroll
            for (int u = 0; u < 8; ++u) top = fmaxf(top, fabsf(v[u]));
          }
        const int ex = (top > 0.f && top <= 3.402823466e38f) ? 13 - ilogbf(top) : 0;
        crow = scalbnf(a.scale * kLog2e, -ex);
        const float fa = scalbnf(1.f, ex / 2), fb = scalbnf(1.f, ex - ex / 2);     // (each a normal number)
        uint8_t* qrow = smem + t * C::kTileBytes + r * 128;
#pragma unroll
        for (int f = 0; f < D; f += 8) {
          uint4 p = make_uint4(0u, 0u, 0u, 0u);
          if (row_ok && f < cc.d) {
            float v[8];
            load8(f, v);
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = v[u] * fa * fb;
            p = make_uint4(pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3]), pack2<false>(v[4], v[5]), pack2<false>(v[6], v[7]));
          }
          *reinterpret_cast<uint4*>(qrow + (f / 64) * kChunkBytes + ((((f / 8) & 7) ^ (r & 7)) << 4)) = p;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->q_full[t]);
      }

      // Where this thread's row has its partial results in the workspace: (maximum, sum) and, behind all of these, outputs.  What
      // tensor memory had summed up so far is there, too, with the maximum that it refers to.  (The row is worked out anew, so that
      // nothing of it lives in registers beside a score row.)
      struct Part {
        float *ml, *o;
        int row, i, hq;
        long long unit;
      };
      auto part = [&]() {
        int tid = threadIdx.x;
        asm volatile("" : "+r"(tid));
        Part p;
        p.row = row0 + ((tid - 128) & 255);
        const int r = p.row < rows ? p.row : 0;
        p.i = r / G;
        p.hq = h * G + r % G;
        p.unit = p.hq + (long long)a.Hq * b;
        const long long at = (p.unit * splits + split) * a.L + p.i;
        p.ml = a.ws + at * 2;
        p.o = a.ws + ((((long long)a.Hq * cc.B * splits * a.L * 2) + 3) & ~3LL) + at * cc.d;
        return p;
      };
      // what such sums are multiplied by beside a maximum that has grown to m
      auto since = [](float then, float m) { return then == m ? 1.f : ex2_approx(then - m); };

      float m_used = neg_inf(), l = 0.f;
      bool ok = true;
      // (a loop around the loop over the tiles: a step that is rarely taken inside it costs its code 4 % and more)
#pragma unroll 1
      for (int j_from = 0; j_from < nt && ok; j_from += kFold) {
        if (j_from > 0) {
          // the products of the tiles so far are done when the scores of the next one are; that one's begin the sums anew
          ok = mbar_wait(&bars->s_full[t], 0, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (!idle) {
            const Part p = part();
            const bool row_ok = p.row < rows, more = j_from > kFold;
            float f = 0.f;
            if (row_ok) {
              if (more) f = since(p.ml[0], m_used);
              p.ml[0] = m_used;
            }
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                if (!row_ok || c * 32 + e >= cc.d) continue;
                float4* to = reinterpret_cast<float4*>(p.o + c * 32 + e);
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
                if (more) s = *to;
                s.x = fmaf(s.x, f, __uint_as_float(o[e]));
                s.y = fmaf(s.y, f, __uint_as_float(o[e + 1]));
                s.z = fmaf(s.z, f, __uint_as_float(o[e + 2]));
                s.w = fmaf(s.w, f, __uint_as_float(o[e + 3]));
                *to = s;
              }
            }
          }
        }
        const int j_to = min(nt, j_from + kFold);
#pragma unroll 1
        for (int j = j_from; j < j_to; ++j) {
          uint8_t* sm = smem;
          asm volatile("" : "+l"(sm));         // (no barrier's address in a register for good)
          BarsC* bb = reinterpret_cast<BarsC*>(sm + C::kBarOff);
          volatile int* abort_flag = &bb->abort_flag;
          if ((j & 3) == 0) ok = mbar_wait_warp(&bb->meta_full[(j >> 2) & 1], (j >> 3) & 1, abort_flag);
          if (!ok) break;
          // scales: a group of SG keys has a factor and an offset
          const PageMeta* pm = reinterpret_cast<const PageMeta*>(sm + C::kMetaOff) + (j & (kMetaTiles - 1)) * 8;
          ok = mbar_wait(&bb->s_full[t], j & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (idle) {
            if (lane == 0) {
              mbar_arrive(&bb->p_half[t][0]);
              mbar_arrive(&bb->p_half[t][1]);
            }
            continue;
          }
          // Twice over the scores, 64 keys at a time: once for the maximum, once for the weights, which overwrite them.  (Held
          // whole in registers, as the 16-bit forward does, a row leaves none for the converting warps, and the longer code
          // keeps every warp waiting for instructions: 2.56 ms when this form took 2.34, 4096 queries over 8192 tokens of 4 sequences.)
          const int j0 = (j_lo + j) * kBN;
          const bool edge = __any_sync(0xffffffffu, j0 + kBN - 1 > lim);
          constexpr int HG = 64 / SG;             // scales of 64 keys
          uint32_t sr[2][32];
          auto fetch = [&](int hf) {
            tmem_ld32(tS + hf * 64, sr[0]);
            tmem_ld32(tS + hf * 64 + 32, sr[1]);
            tmem_wait_ld();
            if (edge) {
              // the scaled logits themselves, -Inf where the row does not look
#pragma unroll
              for (int g = 0; g < HG; ++g) {
                const float f = crow * pm[hf * 4 + g * (SG / 16)].ks, o = pm[hf * 4 + g * (SG / 16)].lvs;
#pragma unroll
                for (int e = g * SG; e < (g + 1) * SG; ++e) {
                  const float v = fmaf(__uint_as_float(sr[e / 32][e & 31]), f, o);
                  sr[e / 32][e & 31] = j0 + hf * 64 + e > lim ? 0xff800000u : __float_as_uint(v);
                }
              }
            }
          };
          auto factor = [&](int hf, int g) { return edge ? 1.f : crow * pm[hf * 4 + g * (SG / 16)].ks; };
          auto offset = [&](int hf, int g) { return edge ? 0.f : pm[hf * 4 + g * (SG / 16)].lvs; };

          float mx = neg_inf();
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {
            fetch(hf);
#pragma unroll
            for (int g = 0; g < HG; ++g) {
              float m0 = neg_inf(), m1 = neg_inf();
#pragma unroll
              for (int e = g * SG; e < (g + 1) * SG; e += 4) {
                m0 = max3(m0, __uint_as_float(sr[e / 32][e & 31]), __uint_as_float(sr[e / 32][(e & 31) + 1]));
                m1 = max3(m1, __uint_as_float(sr[e / 32][(e & 31) + 2]), __uint_as_float(sr[e / 32][(e & 31) + 3]));
              }
              mx = fmaxf(mx, fmaf(fmaxf(m0, m1), factor(hf, g), offset(hf, g)));
            }
          }
          const float m_new = fmaxf(m_used, mx - kBits);
          const bool raise = m_new > m_used + kGap;      // also true for m_used = -Inf < m_new
          if (__any_sync(0xffffffffu, raise)) {
            if (j > 0) {
              const float f = raise ? ex2_approx(m_used - m_new) : 1.f;
              l *= f;
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(tO + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st32(tO + c * 32, o);
              }
            }
            if (raise) m_used = m_new;
          }
          const float ref = m_used == neg_inf() ? 0.f : m_used;
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {
            fetch(hf);
            uint32_t pk[32];
#pragma unroll
            for (int g = 0; g < HG; ++g) {
              const unsigned long long f2 = pair_of(factor(hf, g)), c2 = pair_of(offset(hf, g) - ref);
              unsigned long long s2[2] = {0ull, 0ull};
#pragma unroll
              for (int e = g * SG; e < (g + 1) * SG; e += 2) {
                float x0, x1;
                fma2(x0, x1, __uint_as_float(sr[e / 32][e & 31]), __uint_as_float(sr[e / 32][(e & 31) + 1]), f2, c2);
                x0 = ex2_approx(x0);
                x1 = ex2_approx(x1);
                add2(s2[(e >> 1) & 1], x0, x1);
                pk[e >> 1] = pack2<false>(x0, x1);
              }
              // a page that the row does not see adds nothing, whatever its scale is
              const float sum = pair_sum(s2[0]) + pair_sum(s2[1]);
              if (!(sum == 0.f)) l = fmaf(sum, pm[hf * 4 + g * (SG / 16)].ivs, l);
            }
            tmem_st32(tS + hf * 32, pk);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bb->p_half[t][hf]);
          }
        }
      }

      // -------------------------------------------------- epilogue
      if (ok && nt > 0) {
        ok = mbar_wait(&bars->o_full[t], 0, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
      }
      if (ok) {
        tc_fence_after();
        const bool dead = l == 0.f;
        const Part p = part();
        const bool row_ok = p.row < rows, folded = nt > kFold;
        float f_since = 0.f;
        if (folded && row_ok) f_since = since(p.ml[0], m_used);
        T* xrow = nullptr;
        float inv = 1.f;
        if (splits > 1) {
          if (row_ok) {
            p.ml[0] = m_used - kBits;              // (l has that factor)
            p.ml[1] = l;
          }
        } else {
          xrow = reinterpret_cast<T*>(a.x) + (long long)p.i * a.x_sl + (long long)b * a.x_sb + (long long)p.hq * cc.d;
          inv = dead ? (a.nan_fm ? __int_as_float(0x7fc00000) : 0.f) : 1.f / l;
          if (row_ok && a.lse) a.lse[p.i + (long long)a.L * p.unit] = dead ? neg_inf() : (m_used - kBits + log2f(l)) * kLn2;
        }
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (nt > 0) {
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (!row_ok || c * 32 + e >= cc.d) continue;
            float f[8];
            if (folded) {
#pragma unroll
              for (int u = 0; u < 8; ++u) o[e + u] = __float_as_uint(fmaf(p.o[c * 32 + e + u], f_since, __uint_as_float(o[e + u])));
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) f[u] = dead ? (splits > 1 ? 0.f : inv) : __uint_as_float(o[e + u]) * inv;
            if (splits > 1) {
              *reinterpret_cast<float4*>(p.o + c * 32 + e) = make_float4(f[0], f[1], f[2], f[3]);
              *reinterpret_cast<float4*>(p.o + c * 32 + e + 4) = make_float4(f[4], f[5], f[6], f[7]);
            } else if (vec) {
              *reinterpret_cast<uint4*>(xrow + c * 32 + e) =
                  make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7]));
            } else {
#pragma unroll
              for (int u = 0; u < 8; ++u) xrow[c * 32 + e + u] = Elem<T>::from_f(f[u]);
            }
          }
        }
      }
    }
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) {
    atomicExch(&g_cache_attn_abort, 1);
    if (a.status) atomicExch(a.status, NNLIB_B200_TIMEOUT);
  }
}

template <typename T, int D, int CODE, int SG>
cudaError_t launch(const CacheAttnArgs& a, int splits, cudaStream_t st) {
  const long long rows = (long long)a.L * (a.Hq / a.c.H);
  const long long blocks = (rows + kTiles * kBM - 1) / (kTiles * kBM) * a.c.B * a.c.H * splits;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const bool vec = aligned16(a.q) && aligned16(a.x) && a.q_sl % 8 == 0 && a.q_sb % 8 == 0 && a.x_sl % 8 == 0 && a.x_sb % 8 == 0;
  auto kernel = cache_attn_umma_kernel<T, D, CODE, SG>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, CfgC<D>::kSmemBytes);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)blocks, kThreadsC, CfgC<D>::kSmemBytes, st>>>(a, splits, vec ? 1 : 0);
  count_launch();
  return cudaGetLastError();
}

template <typename T, int CODE>
cudaError_t launch_d(const CacheAttnArgs& a, int splits, cudaStream_t st) {
  if (a.c.log_page >= 6) return a.c.d <= 64 ? launch<T, 64, CODE, 64>(a, splits, st) : launch<T, 128, CODE, 64>(a, splits, st);
  return a.c.d <= 64 ? launch<T, 64, CODE, 16>(a, splits, st) : launch<T, 128, CODE, 16>(a, splits, st);
}

template <typename T>
cudaError_t launch_c(const CacheAttnArgs& a, int splits, cudaStream_t st) {
  return a.c.code == NNLIB_B200_INT8 ? launch_d<T, NNLIB_B200_INT8>(a, splits, st) : launch_d<T, NNLIB_B200_E4M3>(a, splits, st);
}

// keys of a sequence at most
long long most_keys(const CacheAttnArgs& a) {
  const long long cap = a.c.rows << a.c.log_page;
  return a.lens ? cap : std::min(cap, std::max(a.len0, 0LL));
}

}  // namespace

bool cache_umma_supports(const CacheAttnArgs& a, int dtype) { return dtype != NNLIB_B200_F32 && a.c.d <= 128; }

// Blocks of keys of a unit: where there are too few blocks of rows to fill the GPU, with four tiles of keys each at least.
// What the host knows of the lengths is the capacity, or len0.
int cache_umma_splits(const CacheAttnArgs& a) {
  const long long rows = (long long)a.L * (a.Hq / a.c.H);
  const long long blocks = (rows + kTiles * kBM - 1) / (kTiles * kBM) * a.c.B * a.c.H;
  const long long n = std::min(148 / std::max(blocks, 1LL), most_keys(a) / (4 * kBN));
  return (int)std::max(1LL, std::min(n, 64LL));
}

// Does a block have, or may it have, partial results in the workspace?
bool cache_umma_parts(const CacheAttnArgs& a, int dtype, int splits) {
  const long long tiles = ((most_keys(a) + kBN - 1) / kBN + splits - 1) / splits;
  return splits > 1 || tiles > (dtype == NNLIB_B200_F16 ? kFoldTiles<__half> : kFoldTiles<__nv_bfloat16>);
}

cudaError_t cache_umma(const CacheAttnArgs& a, int dtype, int splits, cudaStream_t st) {
  return dtype == NNLIB_B200_F16 ? launch_c<__half>(a, splits, st) : launch_c<__nv_bfloat16>(a, splits, st);
}

cudaError_t cache_umma_take_abort(int* out, cudaStream_t st) {
  int v = 0;
  cudaError_t e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return e;
  e = cudaMemcpyFromSymbol(&v, g_cache_attn_abort, sizeof(int));
  if (e != cudaSuccess) return e;
  if (v) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_cache_attn_abort, &zero, sizeof(int));
  }
  *out = v;
  return e;
}

}  // namespace nb200
