// Attention over the 8-bit cache by streamed warp-level products: generated tokens, short runs of them, Float32 arrays.
//
// A key or value element is code * scale, the scale one number per page and head, so both products run on the codes
// themselves, which 16-bit floating point holds exactly:
//   logit_ij = (q_i . kcode_j) * scale * ks(page of j)
//   x_i = sum_j w_ij vcode_j / sum_j w_ij / vs(page of j),   w_ij = 2^(log2e * logit_ij + log2 vs(page of j) - m_i)
// i.e. a page's value scale goes into the exponent, where the running maximum m_i takes it up: no product is scaled, no
// accumulator has a page's scale in it, and a weight's size is the size of what it adds to x.  q_i is brought to a
// largest element in [2^13, 2^14) by a power of two of its own; w is rounded to 16 bits after a factor of 2^14, so that
// weights keep 11 bits down to 2^-28 of the largest.  Float32 arrays: q and w as the sum of two 16-bit terms
// each, sums over the keys by rounded additions (over 246 random shapes 7.4e-7 off at most instead of 2.3e-5; one query each, 32 / 8
// heads of 128, 16 sequences of 8192 tokens, Int8 84.6 us, E4M3 86.3, 1 % and 5 % more than without; 256 queries of 4 sequences
// of 8192, 16 / 4 heads of 64, 555 us).
//
// HBM is the bound (2 d bytes per key and head for up to 16 rows), so what counts is bytes in flight: nothing is staged,
// a warp streams 16 keys at a time straight into the fragments of m16n8k16 products.  Keys and the features of values are
// the products' sixteen rows, queries their eight columns, so that one query costs half of what it would as a row:
//   S^T = K Q^T   lane (g, c) = (lane / 4, lane % 4) takes 16 consecutive features 64 G + 16 c .. of keys g and g + 8: word t
//                 of 16 bytes is what it owes to k-step t, two codes to each register; Q's fragments in the same order.
//   O^T += V^T W^T  rows may be any features: rows g and g + 8 of product j are features g (D/8) + 2j and the next, so a lane
//                 loads D/8 consecutive bytes of each of its four keys 2c, 2c+1, 2c+8, 2c+9 and pairs the codes of two keys
//                 up.  W^T comes from S^T's layout by transposing 8 x 8 blocks.
// The products' additions cut off instead of rounding, by up to 2^-23 of the sum behind sixteen keys.  So a warp of a 16-bit
// call adds what it has to its part of shared memory, rounded, every 32768 keys, which leaves 2^-12 however long the history
// is (nine sequences of 1048576 tokens, a team to each: Float16 1.5e-3 off before).
// Columns: the query heads of a group and the queries, column r = query r / G, head r % G of the group; NT blocks of eight.
// Int8 to 16 bits: (code ^ 0x80) under 0x64 is 1024 + 128 + code, less 1152.  E4M3: the conversion instruction.
// Lengths are known on the device only, and a block more than fit at once costs a second wave.  So the blocks, as many as
// fit, form teams of one for each cache head (what runs at one time then reads whole rows of the cache), and the keys of all
// sequences and tiles of columns, laid end to end in groups of one step of the block's four warps, are dealt to the teams in
// equal runs.  A tile that one team has whole it also finishes; of others each team leaves running maxima, sums and outputs,
// two pieces at most (its first tile's and its last one's), and cache_merge_kernel merges what a tile's first team says
// there is.  (Runs cut so that none reaches into a second tile, where tiles are few: 8 x 1024 tokens 16 us instead of 20, but 8 x
// 8192 43 instead of 42 and 4 x 131072 218 instead of 212, for the registers that it takes.)  One query each, 32 / 8 heads of 128,
// Int8: 4 sequences of 131072 tokens 206 us, 5.2 TB/s; 8 of 8192 42 to 43 us, of which some 14 are the way to the first keys, the
// end and the merging, and 2.8 each step at 5 TB/s; 64 of 2048 71 to 73 us (each sequence's keys cut into parts by themselves: 86).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "cache_codes.cuh"
#include "split_reduce.cuh"

namespace nb200 {
namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kValueFloor = 7.8886090522101181e-31f;    // 2^-100
constexpr float kWeightBits = 14.f;

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float qnan() { return __int_as_float(0x7fc00000); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  uint32_t u;
  memcpy(&u, &v, 4);
  return u;
}

// two codes in the low bytes of the halves of u (as they are: int8) to two 16-bit numbers
__device__ __forceinline__ uint32_t int8_pair(uint32_t biased, uint32_t sel) {
  const uint32_t v = __byte_perm(biased, 0x64646464u, sel);
  uint32_t r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t two) {
  uint32_t r;
  asm("{ .reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t; }" : "=r"(r) : "r"(two));
  return r;
}
// bytes 0, 1 and 2, 3 of a word as two pairs
template <int CODE>
__device__ __forceinline__ void word_pairs(uint32_t w, uint32_t& p0, uint32_t& p1) {
  if (CODE == NNLIB_B200_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    p0 = int8_pair(u, 0x4140u);
    p1 = int8_pair(u, 0x4342u);
  } else {
    p0 = e4m3_pair(w);
    p1 = e4m3_pair(w >> 16);
  }
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 block of 16-bit values: row i / columns 2j, 2j + 1 in lane 4i + j becomes column i / rows 2j, 2j + 1
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// BYTES codes of a lane, as words
template <int BYTES>
__device__ __forceinline__ void load_codes(const unsigned char* p, uint32_t* w) {
  static_assert(BYTES == 8 || BYTES == 16, "one load");
  if constexpr (BYTES == 8)
    asm("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  else
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
}

// The features of a value row that lane group g of eight takes, D / 8 of them, in loads of at most 16: whether it makes its
// load number i for a head of d features (a multiple of 16, at most D, which need not be one of D / 8).
template <int D>
struct ValueLoads {
  static constexpr int kLane = D / 8, kBytes = kLane < 16 ? kLane : 16, kLoads = kLane / kBytes;
  __host__ __device__ static constexpr bool made(int d, int g, int i) { return kLane * g + kBytes * i < d; }
  // every feature of a head is loaded and none behind it
  static constexpr bool exact() {
    for (int d = 16; d <= D; d += 16) {
      int n = 0;
      for (int g = 0; g < 8; ++g)
        for (int i = 0; i < kLoads; ++i)
          if (made(d, g, i)) {
            if (kLane * g + kBytes * (i + 1) > d) return false;
            n += kBytes;
          }
      if (n != d) return false;
    }
    return true;
  }
};
static_assert(ValueLoads<64>::exact() && ValueLoads<128>::exact() && ValueLoads<256>::exact(), "loads of value rows stay in their head");

__device__ __forceinline__ int seq_len(const CacheAttnArgs& a, int b) {
  const long long cap = a.c.rows << a.c.log_page;
  const long long n = a.lens ? (long long)a.lens[b] : a.len0;
  return (int)(n < 0 ? 0 : (n < cap ? n : cap));
}
// position of query 0 of a sequence of len tokens
__device__ __forceinline__ long long seq_start(const CacheAttnArgs& a, int b, int len) {
  return a.start ? (long long)a.start[b] : (long long)len - a.L;
}
// the last key that query i sees
__device__ __forceinline__ int last_key(const CacheAttnArgs& a, long long start, int i, int len) {
  if (!a.causal) return len - 1;
  const long long e = start + i;
  return e < 0 ? -1 : (e < len ? (int)e : len - 1);
}

// KG: sixteens of keys that a warp takes at a time, two where registers allow (what a step costs beside its products is then
// shared); blocks of an SM: as many as do not spill the codes in flight
template <typename T, int D, int NT>
struct Cfg {
  static constexpr int kKG = sizeof(T) == 2 && NT == 1 && D <= 128 ? 2 : 1;
  static constexpr int kCtas = D <= 64 ? 4 : (D <= 128 ? 3 : 2);
};

// a / b, in 32 bits where they do (a division of 64 costs some 500 cycles, which a short call notices)
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ long long share_of(long long total, int i, int n) { return quotient(total * i, n); }

// the sequence, tile of columns and keys that tile number v of a call stands for
struct TileKeys {
  int b, row0, len, kend;
  long long start;
};
__device__ __forceinline__ TileKeys tile_keys(const CacheAttnArgs& a, int v, int tiles, int width, int rows, int G) {
  TileKeys t;
  t.b = v / tiles;
  t.row0 = (v - t.b * tiles) * width;
  t.len = seq_len(a, t.b);
  t.start = seq_start(a, t.b, t.len);
  t.kend = last_key(a, t.start, (min(t.row0 + width, rows) - 1) / G, t.len) + 1;
  return t;
}

// Workspace: (maximum, sum) of 2 * teams pieces, H heads, `width` columns, their outputs, and for each tile of columns the
// first piece's number and how many there are (1: finished, 0: no keys).
__host__ __device__ inline long long piece_slots(int teams, int H, int width) { return 2LL * teams * H * width; }

// T: element type of q and x; HILO: two 16-bit terms for an element of q and for a weight (T = float)
template <typename T, int D, int CODE, int NT>
__global__ void __launch_bounds__(kWarps * 32, Cfg<T, D, NT>::kCtas)
cache_attn_kernel(const CacheAttnArgs a, const int teams, const int vec) {
  constexpr bool HILO = sizeof(T) == 4;
  constexpr int ROWS = 8 * NT, KS = D / 16, GK = D / 64, VB = D / 8, HL = HILO ? 2 : 1, KG = Cfg<T, D, NT>::kKG, kStep = 16 * KG;
  constexpr int GS = kWarps * kStep;             // keys of a group
  __shared__ float sm_o[kWarps][ROWS][D];
  __shared__ float sm_m[kWarps][ROWS], sm_l[kWarps][ROWS];
  __shared__ long long sm_sum[kWarps], sm_base;
  __shared__ int sm_tile;
  const CacheArgs& cc = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int G = a.Hq / cc.H, rows = a.L * G, tiles = (rows + ROWS - 1) / ROWS, n_tiles = tiles * cc.B;
  const int h = blockIdx.x % cc.H, team = blockIdx.x / cc.H;
  float* const ws_o = a.ws + 2 * piece_slots(teams, cc.H, ROWS);
  int2* const ws_meta = reinterpret_cast<int2*>(ws_o + piece_slots(teams, cc.H, ROWS) * cc.d);

  // this team's run of groups: lo .. hi - 1 of all of them, from tile v on, whose first group is number base
  long long lo, hi, total, base;
  int v, n_teams;
  if (a.ws == nullptr) {                         // short sequences: a team for each tile, which has it whole
    v = n_teams = team;
    lo = base = 0;
    hi = total = 1;
  } else {
    const int per = (n_tiles + kWarps * 32 - 1) / (kWarps * 32), v0 = min((int)threadIdx.x * per, n_tiles), v1 = min(v0 + per, n_tiles);
    long long mine = 0;
    for (int i = v0; i < v1; ++i) {
      const int n = (tile_keys(a, i, tiles, ROWS, rows, G).kend + GS - 1) / GS;
      if (n == 0 && blockIdx.x == 0) ws_meta[i] = make_int2(0, 0);
      mine += n;
    }
    long long upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += t;
    }
    if (lane == 31) sm_sum[warp] = upto;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += sm_sum[w];
      total += sm_sum[w];
    }
    n_teams = (int)min((long long)teams, total);
    // (the merging blocks may take their places: all of this grid's have theirs)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (team >= n_teams) return;
    lo = share_of(total, team, n_teams);
    hi = share_of(total, team + 1, n_teams);
    if (upto - mine <= lo && lo < upto) {
      long long at = upto - mine;
      int i = v0;
      for (;; ++i) {
        const int n = (tile_keys(a, i, tiles, ROWS, rows, G).kend + GS - 1) / GS;
        if (lo < at + n) break;
        at += n;
      }
      sm_tile = i;
      sm_base = at;
    }
    __syncthreads();
    v = sm_tile;
    base = sm_base;
  }

  for (bool first = true;; ++v) {
    const TileKeys tk = tile_keys(a, v, tiles, ROWS, rows, G);
    const int n_groups = (tk.kend + GS - 1) / GS;
    if (a.ws == nullptr) hi = n_groups;
    else if (n_groups == 0) continue;
    const int b = tk.b, row0 = tk.row0, len = tk.len, kend = tk.kend;
    const long long start = tk.start;
    const int g_lo = (int)max(lo - base, 0LL), g_hi = (int)min(hi - base, (long long)n_groups);
    const int key_lo = g_lo * GS, key_hi = min(g_hi * GS, kend);
    const unsigned char* kbase = cc.codes[0] + (long long)h * cc.d + 16 * c + g * cc.row;
    const unsigned char* vbase = cc.codes[1] + (long long)h * cc.d + VB * g + 2 * c * cc.row;

    // Pages, 32 sixteens of keys at a time: the warp's sixteen number n (of its steps, one after the other) by lane n
    const int stride = kWarps * kStep;
    int key0 = key_lo + warp * kStep;
    int pg = 0;
    float ksc = 0.f, vsc = 0.f;
    auto look_up = [&](int first) {
      const int key = first + (lane / KG) * stride + (lane % KG) * 16;
      const bool in = key < key_hi;
      const long long page = in ? cache_page(cc, b, (long long)key >> cc.log_page) : -1;
      pg = page < 0 ? 0 : (int)page;
      ksc = page < 0 ? qnan() : cc.scale[0][page * cc.H + h];
      vsc = page < 0 ? qnan() : cc.scale[1][page * cc.H + h];
    };
    uint32_t kf[KG][2][GK][4], vf[KG][4][VB / 4];
    const int T1 = (1 << cc.log_page) - 1;
    const int row8 = 8 * (int)cc.row;
    long long at[KG];                                // where the sixteens of the step under way begin
    auto place = [&](int key, int n) {
#pragma unroll
      for (int kg = 0; kg < KG; ++kg) {
        const int page = __shfl_sync(0xffffffffu, pg, (n * KG + kg) & 31);
        at[kg] = (((long long)page << cc.log_page) + ((key + 16 * kg) & T1)) * cc.row;
      }
    };
    // (a step may reach behind the block's last key, onto a page that is not looked up: page 0 then)
    auto load_k = [&]() {
#pragma unroll
      for (int kg = 0; kg < KG; ++kg) {
        const unsigned char* p = kbase + at[kg];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int G4 = 0; G4 < GK; ++G4)
            if (64 * G4 + 16 * c < cc.d) load_codes<16>(p + nt * row8 + 64 * G4, kf[kg][nt][G4]);
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int kg = 0; kg < KG; ++kg) {
        const unsigned char* p = vbase + at[kg];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int i = 0; i < ValueLoads<D>::kLoads; ++i)
            if (ValueLoads<D>::made(cc.d, g, i))
              load_codes<ValueLoads<D>::kBytes>(p + (u & 1) * (int)cc.row + (u >> 1) * row8 + 16 * i, vf[kg][u] + 4 * i);
      }
    };
#pragma unroll
    for (int kg = 0; kg < KG; ++kg) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int G4 = 0; G4 < GK; ++G4)
#pragma unroll
          for (int w = 0; w < 4; ++w) kf[kg][nt][G4][w] = 0u;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int w = 0; w < VB / 4; ++w) vf[kg][u][w] = 0u;
    }
    // the first keys are on their way while Q is prepared
    if (key0 < key_hi) {
      look_up(key0);
      place(key0, 0);
      load_k();
      load_v();
    }

    // Q's fragments, brought to a largest element in [2^13, 2^14)
    uint32_t qb[NT][HL][KS][2];
    float crow[NT][2];                           // what a column's products are multiplied by, but for the page's scale
    int lim[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = row0 + 8 * t + g, i = row / G, hq = h * G + row % G;
      const bool live = row < rows;
      const T* qp = reinterpret_cast<const T*>(a.q) + (live ? (long long)i * a.q_sl + (long long)b * a.q_sb + (long long)hq * cc.d : 0) + 16 * c;
      float top = 0.f, q[GK][16];
#pragma unroll
      for (int G4 = 0; G4 < GK; ++G4) {
        if (live && 64 * G4 + 16 * c < cc.d) {
          if (vec) {
#pragma unroll
            for (int w = 0; w < (int)sizeof(T); ++w) {
              constexpr int U = 16 / sizeof(T);
              const uint4 raw = __ldg(reinterpret_cast<const uint4*>(qp + 64 * G4) + w);
              T e[U];
              memcpy(e, &raw, 16);
#pragma unroll
              for (int u = 0; u < U; ++u) q[G4][w * U + u] = Elem<T>::to_f(e[u]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) q[G4][e] = Elem<T>::to_f(qp[64 * G4 + e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) q[G4][e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(q[G4][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int ex = (top > 0.f && top <= 3.402823466e38f) ? 13 - ilogbf(top) : 0;
      const float cr = scalbnf(a.scale * kLog2e, -ex);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        crow[t][u] = __shfl_sync(0xffffffffu, cr, 4 * (2 * c + u));
        const int mine = row0 + 8 * t + 2 * c + u;
        lim[t][u] = mine < rows ? last_key(a, start, mine / G, len) : -1;
      }
      // a power of two in two factors, each a normal number
      const float fa = scalbnf(1.f, ex / 2), fb = scalbnf(1.f, ex - ex / 2);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = q[ks / 4][4 * (ks % 4) + e] * fa * fb;
        qb[t][0][ks][0] = half2_bits(v[0], v[1]);
        qb[t][0][ks][1] = half2_bits(v[2], v[3]);
        if constexpr (HILO) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] -= __half2float(__float2half_rn(v[e]));
          qb[t][1][ks][0] = half2_bits(v[0], v[1]);
          qb[t][1][ks][1] = half2_bits(v[2], v[3]);
        }
      }
    }

    float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int u = 0; u < 2; ++u) m[t][u] = ninf(), l[t][u] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][j][e] = 0.f;
    }

    int lim_all = 0x7fffffff;                    // up to here every column of the tile sees every key
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) lim_all = min(lim_all, lim[t][u]);
    lim_all = __reduce_min_sync(0xffffffffu, lim_all);

    // Products' additions cut off (below), so a warp of a 16-bit call sums up 32768 keys by them; what it has is then added,
    // rounded, to its part of shared memory, with the maximum that it refers to, and begun anew.
    constexpr int kFold = 32768 / kStep;
    auto since = [](float then, float now) { return then == now ? 1.f : ex2(then - now); };
    int n = 0;
    for (;;) {
      const int key_stop = HL == 1 && key_hi - key0 > kFold * stride ? key0 + kFold * stride : key_hi;
      for (; key0 < key_stop; key0 += stride, ++n) {
        float ks[KG], vs[KG];
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
          ks[kg] = __shfl_sync(0xffffffffu, ksc, (n * KG + kg) & 31);
          vs[kg] = __shfl_sync(0xffffffffu, vsc, (n * KG + kg) & 31);
        }
        const int next = key0 + stride;
        if (next < key_hi) {
          if (((n + 1) * KG & 31) == 0) look_up(next);
          place(next, n + 1);
        }

        float sc[KG][NT][4];
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[kg][t][e] = 0.f;
#pragma unroll
          for (int k2 = 0; k2 < KS; ++k2) {
            uint32_t a0, a1, a2, a3;
            word_pairs<CODE>(kf[kg][0][k2 / 4][k2 % 4], a0, a2);
            word_pairs<CODE>(kf[kg][1][k2 / 4][k2 % 4], a1, a3);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int hl = 0; hl < HL; ++hl) mma(sc[kg][t], a0, a1, a2, a3, qb[t][hl][k2][0], qb[t][hl][k2][1]);
          }
        }
        if (next < key_hi) load_k();

        // scales of this step's pages (sixteen keys never cross one)
        float lvs[KG], ivs[KG];
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
          const float vse = vs[kg] >= kValueFloor ? vs[kg] : ((vs[kg] >= 0.f) ? kValueFloor : qnan());
          lvs[kg] = __log2f(vse) + kWeightBits;
          ivs[kg] = __fdividef(1.f, vse);
        }
        const bool edge = key0 + kStep - 1 > lim_all;
        uint32_t pb[KG][NT][HL][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          // w[.][e]: key g (+ 8 for e >= 2), column 2c (+ 1 for odd e)
          float w[KG][4];
#pragma unroll
          for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[kg][e] = fmaf(sc[kg][t][e], crow[t][e & 1] * ks[kg], lvs[kg]);
          if (edge) {
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (key0 + 16 * kg + g + (e >> 1) * 8 > lim[t][e & 1]) w[kg][e] = ninf();
          }
          float mn[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float mx = fmaxf(w[0][u], w[0][2 + u]);
            if (KG == 2) mx = fmaxf(mx, fmaxf(w[KG - 1][u], w[KG - 1][2 + u]));
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            mn[u] = fmaxf(m[t][u], mx - kWeightBits);
          }
          if (__any_sync(0xffffffffu, mn[0] > m[t][0] || mn[1] > m[t][1])) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float fo = (m[t][u] == ninf()) ? 0.f : ex2(m[t][u] - mn[u]);
              l[t][u] *= fo;
#pragma unroll
              for (int j = 0; j < D / 16; ++j) {
                o[t][j][u] *= fo;
                o[t][j][2 + u] *= fo;
              }
              m[t][u] = mn[u];
            }
          }
          const float ref[2] = {mn[0] == ninf() ? 0.f : mn[0], mn[1] == ninf() ? 0.f : mn[1]};
#pragma unroll
          for (int kg = 0; kg < KG; ++kg) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[kg][e] = ex2(w[kg][e] - ref[e & 1]);
            // this lane's keys only; a page that the query does not see adds nothing, whatever its scale is
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float sum = w[kg][u] + w[kg][2 + u];
              if (!(sum == 0.f)) l[t][u] = fmaf(sum, ivs[kg], l[t][u]);
            }
#pragma unroll
            for (int hl = 0; hl < HL; ++hl) {
              pb[kg][t][hl][0] = transposed(half2_bits(w[kg][0], w[kg][1]));
              pb[kg][t][hl][1] = transposed(half2_bits(w[kg][2], w[kg][3]));
              if (HILO && hl == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[kg][e] -= __half2float(__float2half_rn(w[kg][e]));
              }
            }
          }
        }
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
          // E4M3 has a NaN; a slot behind the last token may hold anything, and so may page 0, which is read in the place of a
          // page that the pool does not have (its scale is NaN here)
          if (CODE == NNLIB_B200_E4M3 && (key0 + kStep > kend || !(vs[kg] >= 0.f))) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (key0 + 16 * kg + 2 * c + (u & 1) + (u >> 1) * 8 >= kend || !(vs[kg] >= 0.f))
#pragma unroll
                for (int w = 0; w < VB / 4; ++w) vf[kg][u][w] = 0u;
          }
#pragma unroll
          for (int w = 0; w < VB / 4; ++w) {
            // the codes of keys 2c and 2c + 1 side by side, features 4w .. 4w + 3
            const uint32_t a01 = __byte_perm(vf[kg][0][w], vf[kg][1][w], 0x5140), a23 = __byte_perm(vf[kg][0][w], vf[kg][1][w], 0x7362);
            const uint32_t b01 = __byte_perm(vf[kg][2][w], vf[kg][3][w], 0x5140), b23 = __byte_perm(vf[kg][2][w], vf[kg][3][w], 0x7362);
            uint32_t lo[4], hi[4];
            word_pairs<CODE>(a01, lo[0], lo[1]);
            word_pairs<CODE>(a23, lo[2], lo[3]);
            word_pairs<CODE>(b01, hi[0], hi[1]);
            word_pairs<CODE>(b23, hi[2], hi[3]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                if constexpr (HL == 1) {
                  mma(o[t][2 * w + j], lo[2 * j], lo[2 * j + 1], hi[2 * j], hi[2 * j + 1], pb[kg][t][0][0], pb[kg][t][0][1]);
                } else {
                  // The products' own addition cuts off instead of rounding: over a long run the sum shrinks by a part of
                  // 2^-24 a step (2e-5 of x behind 99163 keys).  Float32 sums are added up with rounded additions.
                  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                  for (int hl = 0; hl < HL; ++hl)
                    mma(part, lo[2 * j], lo[2 * j + 1], hi[2 * j], hi[2 * j + 1], pb[kg][t][hl][0], pb[kg][t][hl][1]);
#pragma unroll
                  for (int u = 0; u < 4; ++u) o[t][2 * w + j][u] += part[u];
                }
              }
          }
        }
        if (next < key_hi) load_v();
      }
      if (HL != 1 || key0 >= key_hi) break;
      const bool more = n > kFold;                   // (what the warp put there itself)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = 8 * t + 2 * c + u;
          const float f = more ? since(sm_m[warp][row], m[t][u]) : 0.f;
#pragma unroll
          for (int j = 0; j < D / 16; j += 2) {
            float4* to = reinterpret_cast<float4*>(&sm_o[warp][row][VB * g + 2 * j]);
            const float4 s = more ? *to : make_float4(0.f, 0.f, 0.f, 0.f);
            *to = make_float4(fmaf(s.x, f, o[t][j][u]), fmaf(s.y, f, o[t][j][2 + u]), fmaf(s.z, f, o[t][j + 1][u]), fmaf(s.w, f, o[t][j + 1][2 + u]));
            o[t][j][u] = o[t][j][2 + u] = o[t][j + 1][u] = o[t][j + 1][2 + u] = 0.f;
          }
          __syncwarp();
          if (g == 0) sm_m[warp][row] = m[t][u];
          __syncwarp();
        }
    }
    const bool folded = HL == 1 && n > kFold;

    // merge the four warps
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = 8 * t + 2 * c + u;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[t][u] += __shfl_xor_sync(0xffffffffu, l[t][u], off);
        if (folded) {
          const float f = since(sm_m[warp][row], m[t][u]);
#pragma unroll
          for (int j = 0; j < D / 16; j += 2) {
            const float4 s = *reinterpret_cast<const float4*>(&sm_o[warp][row][VB * g + 2 * j]);
            o[t][j][u] = fmaf(s.x, f, o[t][j][u]);
            o[t][j][2 + u] = fmaf(s.y, f, o[t][j][2 + u]);
            o[t][j + 1][u] = fmaf(s.z, f, o[t][j + 1][u]);
            o[t][j + 1][2 + u] = fmaf(s.w, f, o[t][j + 1][2 + u]);
          }
          __syncwarp();
        }
        if (g == 0) {
          sm_m[warp][row] = m[t][u];
          sm_l[warp][row] = l[t][u];
        }
        // rows g and g + 8 of product j: features VB g + 2j and the next
#pragma unroll
        for (int j = 0; j < D / 16; j += 2)
          *reinterpret_cast<float4*>(&sm_o[warp][row][VB * g + 2 * j]) =
              make_float4(o[t][j][u], o[t][j][2 + u], o[t][j + 1][u], o[t][j + 1][2 + u]);
      }
    __syncthreads();
    const bool whole = g_lo == 0 && g_hi == n_groups;
    const int piece = 2 * team + (first ? 0 : 1);
    if (a.ws != nullptr && g_lo == 0 && h == 0 && threadIdx.x == 0) {
      // the last team of this tile: the last one whose run begins at or before its last group
      const int last = (int)quotient((base + n_groups) * n_teams - 1, total);
      ws_meta[v] = make_int2(piece, last - team + 1);
    }
    for (int idx = threadIdx.x; idx < ROWS * D; idx += kWarps * 32) {
      const int rr = idx / D, e = idx % D, row = row0 + rr;
      if (row >= rows) break;
      const int i = row / G, hq = h * G + row % G;
      float M = ninf(), L = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][rr]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = sm_m[w][rr], f = mw == ninf() ? (sm_l[w][rr] == 0.f ? 0.f : 1.f) : ex2(mw - M);
        L = fmaf(sm_l[w][rr], f, L);
        if (f != 0.f) acc = fmaf(sm_o[w][rr][e], f, acc);
      }
      if (!whole) {
        const long long at = ((long long)piece * cc.H + h) * ROWS + rr;
        if (e < cc.d) ws_o[at * cc.d + e] = acc;
        if (e == 0) *reinterpret_cast<float2*>(a.ws + 2 * at) = make_float2(M, L);
      } else {
        const bool dead = L == 0.f;
        if (e < cc.d) {
          const float out = dead ? (a.nan_fm ? qnan() : 0.f) : acc / L;
          reinterpret_cast<T*>(a.x)[(long long)i * a.x_sl + (long long)b * a.x_sb + (long long)hq * cc.d + e] = Elem<T>::from_f(out);
        }
        if (e == 0 && a.lse) a.lse[i + (long long)a.L * (hq + (long long)a.Hq * b)] = dead ? ninf() : fmaf(M - kWeightBits, 0.6931471805599453f, logf(L));
      }
    }
    first = false;
    base += n_groups;
    if (base >= hi) break;
    __syncthreads();                               // what the warps left has been read
  }
}

// One block for a query and head: merges the pieces of its tile, in order.  Latency is what bounds it: the lanes of a warp take
// a piece each for its maximum, sum and weight, and hand these round while the outputs of eight are under way.
template <typename T>
__global__ void __launch_bounds__(128) cache_merge_kernel(const CacheAttnArgs a, const int teams, const int width) {
  const CacheArgs& cc = a.c;
  const int G = a.Hq / cc.H, rows = a.L * G, tiles = (rows + width - 1) / width, lane = threadIdx.x & 31;
  const int i = blockIdx.x % a.L, unit = blockIdx.x / a.L, hq = unit % a.Hq, b = unit / a.Hq, h = hq / G;
  const int row = i * G + hq - h * G, tile = row / width, r = row - tile * width;
  const float* ws_o = a.ws + 2 * piece_slots(teams, cc.H, width);
  // (launched while the kernel before it ends: its results are there from here on)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 meta = reinterpret_cast<const int2*>(ws_o + piece_slots(teams, cc.H, width) * cc.d)[b * tiles + tile];
  if (meta.y == 1) return;
  T* xrow = reinterpret_cast<T*>(a.x) + (long long)i * a.x_sl + (long long)b * a.x_sb + (long long)hq * cc.d;
  auto at = [&](int k) { return ((long long)(k == 0 ? meta.x : 2 * (meta.x / 2 + k)) * cc.H + h) * width + r; };
  float M = ninf();
  for (int k = lane; k < meta.y; k += 32) {
    const float2 ml = *reinterpret_cast<const float2*>(a.ws + 2 * at(k));
    M = fmaxf(M, ml.x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  for (int e0 = threadIdx.x - lane; e0 < cc.d; e0 += 128) {
    const int e = min(e0 + lane, cc.d - 1);      // (lanes past the end keep their warp company)
    float L = 0.f, acc = 0.f;
    for (int k0 = 0; k0 < meta.y; k0 += 32) {
      const int cnt = min(32, meta.y - k0);
      const float2 ml = *reinterpret_cast<const float2*>(a.ws + 2 * at(k0 + min(lane, cnt - 1)));
      // a piece without a finite maximum is one that no key of was seen, or one with a NaN
      const float f = ml.x == ninf() ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - M);
      for (int j0 = 0; j0 < cnt; j0 += 8) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = ws_o[at(k0 + min(j0 + j, cnt - 1)) * cc.d + e];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float fj = __shfl_sync(0xffffffffu, f, j0 + j), lj = __shfl_sync(0xffffffffu, ml.y, j0 + j);
          // (a sum that is NaN, of a query that sees such a page, counts however small its piece's weight is)
          if (j0 + j < cnt && (fj != 0.f || lj != lj)) {
            L = fmaf(fj, lj, L);
            acc = fmaf(fj, o[j], acc);
          }
        }
      }
    }
    const bool dead = L == 0.f;
    if (e0 + lane < cc.d) xrow[e] = Elem<T>::from_f(dead ? (a.nan_fm ? qnan() : 0.f) : acc / L);
    if (threadIdx.x == 0 && e0 == 0 && a.lse)
      a.lse[i + (long long)a.L * unit] = dead ? ninf() : fmaf(M - kWeightBits, 0.6931471805599453f, logf(L));
  }
}

int row_tile(const CacheAttnArgs& a, int dtype) {
  // (two 16-bit terms, or a head of 256 features, leave registers for eight columns only)
  return (dtype == NNLIB_B200_F32 || a.c.d > 128 || (long long)a.L * (a.Hq / a.c.H) <= 8) ? 8 : 16;
}

// Blocks for each cache head: as many as fit the GPU at once.
int team_count(const CacheAttnArgs& a) {
  const int fit = a.c.d <= 64 ? 4 : (a.c.d <= 128 ? 3 : 2);      // blocks of an SM (Cfg)
  return std::max(1, fit * 148 / a.c.H);
}

// At most 512 tokens to a sequence, and blocks enough for a whole tile each: nothing is merged, one launch and no workspace.
// Measured (us on the device, one launch / dealt out and merged; an eager call, which its caller bounds, 11 and 15): 16-bit, 12
// heads of 64, 1 sequence, 256 tokens 5.5 / 8.4, 512 7.4 / 8.6, 640 8.6 / 8.7, 1024 11.5 / 8.8; 32 / 8 heads of 128, 1 sequence,
// 256 8.5 / 10.6, 512 11.5 / 10.8, 1024 17.5 / 11.2, 8 sequences, 512 11.7 / 12.7, 640 13.1 / 13.4, 1024 17.6 / 20.1; heads
// of 256, 256 12.2 / 12.5, 512 17.1 / 13.0; Float32, heads of 64, 256 6.7 / 7.7, 512 10.0 / 8.3.
bool one_launch(const CacheAttnArgs& a, int dtype) {
  long long cap = a.c.rows << a.c.log_page;
  if (!a.lens) cap = std::min(cap, std::max(a.len0, 0LL));
  const int width = row_tile(a, dtype), rows = a.L * (a.Hq / a.c.H);
  return cap <= 512 && (long long)((rows + width - 1) / width) * a.c.B <= team_count(a);
}

AttnArgs reduce_args(const CacheAttnArgs& a) {
  AttnArgs r;
  std::memset(&r, 0, sizeof(r));
  r.x = a.x;
  r.x_sl = a.x_sl;
  r.x_sb = a.x_sb;
  r.lse = a.lse;
  r.lse_sb = (long long)a.L * a.Hq;
  r.ws = a.ws;
  r.inv_keep = 1.f;
  r.nan_fm = a.nan_fm;
  r.dv = a.c.d;
  r.H = a.Hq;
  r.B = a.c.B;
  r.Lq = a.L;
  return r;
}

// Many columns go to the tensor cores, whose blocks take 256 of them at once but some 12 us to begin: more than 16 columns, and
// more than five groups of keys to a team here.  Measured (us; here / there), 32 / 8 heads of 128: 4 x 16384 tokens, 16 columns
// 67 / 89, 32 99 / 90, 64 177 / 93; 32 x 2048 tokens, 16 columns 74 / 100, 32 129 / 101; 8 / 8 heads, 8 x 4096 tokens, 16
// columns 46 / 53, 24 62 / 55; 16 / 2 heads, 1 x 8192 tokens (3.5 groups) 96 columns 30 / 28, 192 (6.9) 44 / 33; 12 heads of 64,
// 2 x 1000 tokens (1.3 groups), 24 columns 17 / 19.  Where lengths are on the device the capacity stands for them.
bool use_umma(const CacheAttnArgs& a, int dtype) {
  const long long rows = (long long)a.L * (a.Hq / a.c.H);
  if (!cache_umma_supports(a, dtype) || rows <= 16) return false;
  long long cap = a.c.rows << a.c.log_page;
  if (!a.lens) cap = std::min(cap, std::max(a.len0, 0LL));
  return (rows + 15) / 16 * a.c.B * ((cap + 63) / 64) > 5LL * team_count(a);
}

template <typename T>
cudaError_t reduce(const CacheAttnArgs& a, int splits, cudaStream_t st) {
  const AttnArgs r = reduce_args(a);
  attn_split_reduce_kernel<T, false><<<(unsigned)((long long)a.Hq * a.c.B * a.L), 128, 0, st>>>(r, splits);
  count_launch();
  return cudaGetLastError();
}

template <typename T, int D, int CODE, int NT>
cudaError_t launch(const CacheAttnArgs& a, cudaStream_t st) {
  const bool one = a.ws == nullptr;
  const int teams = one ? (a.L * (a.Hq / a.c.H) + 8 * NT - 1) / (8 * NT) * a.c.B : team_count(a);
  const bool vec = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_sl * sizeof(T) % 16 == 0 && a.q_sb * sizeof(T) % 16 == 0;
  cache_attn_kernel<T, D, CODE, NT><<<(unsigned)(teams * a.c.H), kWarps * 32, 0, st>>>(a, teams, vec ? 1 : 0);
  count_launch();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || one) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)a.Hq * a.c.B * a.L));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, cache_merge_kernel<T>, a, teams, 8 * NT);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int CODE>
cudaError_t launch_d(const CacheAttnArgs& a, int rows, cudaStream_t st) {
  if (a.c.d > 128) return launch<T, 256, CODE, 1>(a, st);
  if constexpr (sizeof(T) == 2) {
    if (rows == 16) return a.c.d <= 64 ? launch<T, 64, CODE, 2>(a, st) : launch<T, 128, CODE, 2>(a, st);
  }
  return a.c.d <= 64 ? launch<T, 64, CODE, 1>(a, st) : launch<T, 128, CODE, 1>(a, st);
}

template <typename T>
cudaError_t launch_c(const CacheAttnArgs& a, int rows, cudaStream_t st) {
  return a.c.code == NNLIB_B200_INT8 ? launch_d<T, NNLIB_B200_INT8>(a, rows, st) : launch_d<T, NNLIB_B200_E4M3>(a, rows, st);
}

}  // namespace

bool cache_attn_umma_path(const CacheAttnArgs& a, int dtype) { return use_umma(a, dtype); }

size_t cache_attn_workspace_bytes(const CacheAttnArgs& a, int dtype) {
  if (use_umma(a, dtype)) {
    const int n = cache_umma_splits(a);
    return cache_umma_parts(a, dtype, n) ? sizeof(float) * (size_t)split_ws_floats(reduce_args(a), n) : 0;
  }
  if (one_launch(a, dtype)) return 0;
  const int width = row_tile(a, dtype), rows = a.L * (a.Hq / a.c.H);
  return sizeof(float) * (size_t)(piece_slots(team_count(a), a.c.H, width) * (2 + a.c.d)) +
         sizeof(int2) * (size_t)((rows + width - 1) / width) * a.c.B;
}

cudaError_t cache_attn(CacheAttnArgs a, int dtype, cudaStream_t st) {
  if (use_umma(a, dtype)) {
    const int n = cache_umma_splits(a);
    const cudaError_t e = cache_umma(a, dtype, n, st);
    if (e != cudaSuccess || n == 1) return e;
    return dtype == NNLIB_B200_F16 ? reduce<__half>(a, n, st) : reduce<__nv_bfloat16>(a, n, st);
  }
  if (one_launch(a, dtype)) a.ws = nullptr;
  const int rows = row_tile(a, dtype);
  if (dtype == NNLIB_B200_F16) return launch_c<__half>(a, rows, st);
  if (dtype == NNLIB_B200_BF16) return launch_c<__nv_bfloat16>(a, rows, st);
  return launch_c<float>(a, rows, st);
}

}  // namespace nb200
