// Low-rank adapters of many requests beside one shared projection:
//   y[t] += scale[i] * B_i (A_i x[t]),  i = index[t],
// A [L, R, K], B [L, N, R] in 16 bits, products and sums in float32, y rounded
// once.  Rows whose index is outside [0, L) are not touched.
//
// Tokens of one adapter form tiles of 16 or 64.  Every workgroup finds its own
// tile from the index (up to 4096 tokens: a count per adapter in LDS; above,
// the schedule of ccq_moe_align), then two products run on the matrix cores:
//   shrink  p[t, r] = sum_k x[t, k] A[i, r, k]
//   expand  y[t, n] += sum_r (scale * p[t, r]) B[i, n, r].
// Few tokens: one kernel does both, each workgroup forming p anew for its
// columns.  Else two kernels, p's partial sums (K split over workgroups)
// passing through the workspace and added in the splits' order.
#include "ccq_common.h"

#include <math.h>

namespace ccq {

namespace {

constexpr int LR_THREADS = 512, LR_WAVES = 8;
constexpr int LR_MAX_R = 256;
constexpr int LR_MAX_L = 1024;
constexpr int LR_SELF = 4096;   // most tokens that workgroups sort themselves

struct LoraP {
  const void* x;
  void* y;
  const int64_t* index;
  const void* a;
  const void* b;
  const float* scale;
  const int32_t* rank;
  int32_t* tile_rows;           // [tiles][TM], -1: padding
  int32_t* tile_adapter;        // [tiles], -1: no such tile
  const int32_t* meta;          // tiles of ccq_moe_align's schedule; null: workgroups sort
  float* p;                     // [S][T][Rp]
  int64_t ldx, ldy;
  int T, L, R, Rp, K, N;
  int S, kchunk;                // splits of K, K per split (a multiple of 32)
  int tiles, ncols;             // tiles of the grid, columns per workgroup
  int y_dtype;
};

template <int DT>
struct Half;
template <>
struct Half<CCQ_BF16> {
  using vec = bf16x8;
};
template <>
struct Half<CCQ_F16> {
  using vec = f16x8;
};

__device__ __forceinline__ f32x4 lr_mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 lr_mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 8 values of a row of `len` from element k on, as loaded; past the end 0.
// len % 8 == 0 (uniform): one load at any alignment, of a piece inside the
// row where k is past the end.
template <int DT>
struct Raw {
  u32x4 v[DT == CCQ_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw<DT> lr_load(const void* base, int64_t row, int k, int len) {
  constexpr int E = DT == CCQ_F32 ? 4 : 2;
  Raw<DT> r;
  const char* p = reinterpret_cast<const char*>(base) + row * E;
  if (len % 8 == 0) {
    __builtin_memcpy(&r, p + (int64_t)min(k, len - 8) * E, 8 * E);
  } else if (k + 8 <= len) {
    __builtin_memcpy(&r, p + (int64_t)k * E, 8 * E);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) w[e] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < len) {
        if constexpr (DT == CCQ_F32)
          w[e] = reinterpret_cast<const uint32_t*>(p)[k + e];
        else
          w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[k + e] << (16 * (e & 1));
      }
  }
  return r;
}
template <int DT>
__device__ __forceinline__ Raw<DT> lr_load_whole(const void* base, int64_t row, int k) {
  constexpr int E = DT == CCQ_F32 ? 4 : 2;
  Raw<DT> r;
  __builtin_memcpy(&r, reinterpret_cast<const char*>(base) + (row + k) * E, 8 * E);
  return r;
}
// the values from element n (of 8) on as 0
template <int DT>
__device__ __forceinline__ void lr_mask(Raw<DT>& r, int n) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
  if constexpr (DT == CCQ_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = e < n ? w[e] : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] &= (2 * e < n ? 0xFFFFu : 0u) | (2 * e + 1 < n ? 0xFFFF0000u : 0u);
  }
}
template <int DT>
__device__ __forceinline__ float lr_f32(const Raw<DT>& r, int e) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
  if constexpr (DT == CCQ_F32) return __uint_as_float(w[e]);
  const uint32_t u = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
  return DT == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
}

__device__ __forceinline__ int lr_rank(const LoraP& p, int adapter) {
  return p.rank != nullptr ? min(max(p.rank[adapter], 0), p.R) : p.R;
}

// -------------------------------------------------------------- the tile --
// Tile `tile` of the tokens sorted by adapter (tokens in order within one),
// each adapter's run padded to whole tiles of TM: its adapter (-1: there is no
// such tile) and token ids.  Wave w holds tokens 64 (w CH + c) + lane.
template <int TM>
struct TileS {
  int adapter, first;           // first: the tile's place among its adapter's
  int rows[TM];
};
template <int CH>
struct SortS {
  int count[LR_MAX_L];
  int sum[LR_WAVES];
};

template <int TM, int CH>
__device__ void lr_find_tile(const LoraP& p, int tile, TileS<TM>& t, SortS<CH>& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int key[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = 64 * (wave * CH + c) + lane;
    const int64_t i = at < p.T ? p.index[at] : -1;
    key[c] = i >= 0 && i < p.L ? (int)i : -1;
  }
  for (int i = tid; i < p.L; i += LR_THREADS) s.count[i] = 0;
  if (tid == 0) t.adapter = -1;
  if (tid < TM) t.rows[tid] = -1;
  __syncthreads();
  // a run of equal keys among neighbouring lanes is counted by its first lane
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int before = __shfl_up(key[c], 1, 64);
    const bool head = lane == 0 || before != key[c];
    const uint64_t heads = __ballot(head), behind = lane == 63 ? 0 : heads >> (lane + 1);
    if (head && key[c] >= 0) atomicAdd(&s.count[key[c]], behind ? __builtin_ctzll(behind) + 1 : 64 - lane);
  }
  __syncthreads();
  // tiles before an adapter: each thread takes two neighbouring adapters
  const int n0 = 2 * tid < p.L ? (s.count[2 * tid] + TM - 1) / TM : 0;
  const int n1 = 2 * tid + 1 < p.L ? (s.count[2 * tid + 1] + TM - 1) / TM : 0;
  int sum = n0 + n1;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(sum, off, 64);
    if (lane >= off) sum += v;
  }
  if (lane == 63) s.sum[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += s.sum[w];
  const int start = sum - n0 - n1;
  if (tile >= start && tile < start + n0) {
    t.adapter = 2 * tid;
    t.first = tile - start;
  } else if (tile >= start + n0 && tile < sum) {
    t.adapter = 2 * tid + 1;
    t.first = tile - start - n0;
  }
  __syncthreads();
  const int adapter = t.adapter;
  if (adapter < 0) return;  // uniform
  int mine = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) mine += __popcll(__ballot(key[c] == adapter));
  if (lane == 0) s.sum[wave] = mine;  // the sums of above were read before the last barrier
  __syncthreads();
  int pos = -t.first * TM;
  for (int w = 0; w < wave; ++w) pos += s.sum[w];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint64_t m = __ballot(key[c] == adapter);
    const int at = pos + __popcll(m & ((1ull << lane) - 1));
    if (key[c] == adapter && at >= 0 && at < TM) t.rows[at] = 64 * (wave * CH + c) + lane;
    pos += __popcll(m);
  }
  __syncthreads();
}

// the same from a finished schedule
template <int TM>
__device__ void lr_read_tile(const LoraP& p, int tile, TileS<TM>& t) {
  const bool none = p.meta != nullptr && tile >= p.meta[0];
  if (threadIdx.x < TM) t.rows[threadIdx.x] = none ? -1 : p.tile_rows[(int64_t)tile * TM + threadIdx.x];
  if (threadIdx.x == 0) t.adapter = none ? -1 : p.tile_adapter[tile];
  __syncthreads();
}

// ---------------------------------------------------------------- shrink --
// acc[m][t] += x of rows 16 m + .. times ranks r0 + 16 t + .. over k0 <= k < k1
// (k0 a multiple of 32).  16x16x32 MFMA: A operand lane = token, B operand
// lane = rank, both with k = 8 (lane >> 4) + e (16-bit x and A of one type);
// else the same values in float32 on 16x16x4, element e of every lane in one
// instruction.  Rows and ranks past the end repeat others: not used.
template <int XT, int WT, int MT, int RT>
__device__ __forceinline__ void lr_multiply(const Raw<XT> (&xr)[MT], const Raw<WT> (&ar)[RT], f32x4 (&acc)[MT][RT]) {
  if constexpr (XT == WT) {
    using V = typename Half<WT>::vec;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[m][t] = lr_mfma(__builtin_bit_cast(V, xr[m]), __builtin_bit_cast(V, ar[t]), acc[m][t]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float av = lr_f32<WT>(ar[t], e);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(lr_f32<XT>(xr[m], e), av, acc[m][t], 0, 0, 0);
      }
  }
}

template <int XT, int WT, int MT, int RT>
__device__ __forceinline__ void lr_shrink(const LoraP& p, const int64_t (&xrow)[MT], const int64_t (&arow)[RT], int k0,
                                          int k1, f32x4 (&acc)[MT][RT]) {
  constexpr int U = MT * RT >= 16 ? 1 : MT * RT >= 4 ? 2 : 4;  // k-steps whose loads are in flight together
  const int g = (threadIdx.x >> 4) & 3;
  int k = k0;
  for (; k + 32 * U <= k1 && k + 32 * U <= p.K; k += 32 * U) {
    Raw<XT> xr[U][MT];
    Raw<WT> ar[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int m = 0; m < MT; ++m) xr[u][m] = lr_load_whole<XT>(p.x, xrow[m], k + 32 * u + 8 * g);
#pragma unroll
      for (int t = 0; t < RT; ++t) ar[u][t] = lr_load_whole<WT>(p.a, arow[t], k + 32 * u + 8 * g);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) lr_multiply<XT, WT, MT, RT>(xr[u], ar[u], acc);
  }
  for (; k < k1; k += 32) {
    const int kk = k + 8 * g;
    Raw<XT> xr[MT];
    Raw<WT> ar[RT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m] = lr_load<XT>(p.x, xrow[m], kk, p.K);
#pragma unroll
    for (int t = 0; t < RT; ++t) ar[t] = lr_load<WT>(p.a, arow[t], kk, p.K);
    if (k + 32 > p.K) {
#pragma unroll
      for (int m = 0; m < MT; ++m) lr_mask<XT>(xr[m], p.K - kk);
#pragma unroll
      for (int t = 0; t < RT; ++t) lr_mask<WT>(ar[t], p.K - kk);
    }
    lr_multiply<XT, WT, MT, RT>(xr, ar, acc);
  }
}

// ---------------------------------------------------------------- expand --
// p in parts of the weights' type, most significant first, whose sum is p to
// 16 (two parts of bf16), 24 (three) or 22 bits of the row's largest (two of
// f16, the row scaled by a power of two into its range).
template <int WT, int PARTS>
__device__ __forceinline__ void lr_split(const float (&v)[8], typename Half<WT>::vec (&out)[PARTS]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float rest = v[e];
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      float h;
      if constexpr (WT == CCQ_BF16) {
        const __bf16 b = (__bf16)rest;
        out[i][e] = b;
        h = (float)b;
      } else {
        const _Float16 b = (_Float16)rest;
        out[i][e] = b;
        h = (float)b;
      }
      rest = isfinite(h) ? rest - h : 0.f;
    }
  }
}

// the power of two that brings a row whose largest finite |p| is m into [2^13, 2^14]
__device__ __forceinline__ int lr_exponent(float m) { return m > 0.f ? min(max(13 - ilogbf(m), -100), 100) : 0; }

// Column of D row m of MFMA q in a block of 64: a lane's quads join to 16-byte
// pieces of its token's row, four lanes to 64 contiguous bytes.
template <int YT>
__device__ __forceinline__ int lr_col(int q, int m) {
  return YT == CCQ_F32 ? 16 * q + m : 32 * (q >> 1) + 8 * (m >> 2) + 4 * (q & 1) + (m & 3);
}

// The lane's 16 values of y, block n0 of 64 columns
template <int YT>
struct YBlock {
  static constexpr int PIECES = YT == CCQ_F32 ? 4 : 2, COLS = YT == CCQ_F32 ? 4 : 8;
  u32x4 v[PIECES];
  __device__ __forceinline__ static int col(int piece, int g) { return YT == CCQ_F32 ? 16 * piece + 4 * g : 32 * piece + 8 * g; }
  __device__ __forceinline__ void load(const void* y, int64_t row, int n0, int g, int N) {
    constexpr int E = YT == CCQ_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int n = n0 + col(i, g);
      const char* at = reinterpret_cast<const char*>(y) + (row + n) * E;
      if (n + COLS <= N) {
        __builtin_memcpy(&v[i], at, 16);
      } else {
        v[i] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < COLS; ++e)
          if (n + e < N) {
            if constexpr (YT == CCQ_F32)
              v[i][e] = reinterpret_cast<const uint32_t*>(at)[e];
            else
              v[i][e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(at)[e] << (16 * (e & 1));
          }
      }
    }
  }
  __device__ __forceinline__ void add_store(void* y, int64_t row, int n0, int g, int N, const f32x4 (&acc)[4], float f) {
    constexpr int E = YT == CCQ_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int n = n0 + col(i, g);
      u32x4 o;
      if constexpr (YT == CCQ_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __float_as_uint(__uint_as_float(v[i][e]) + acc[i][e] * f);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4& d = acc[2 * i + (e >> 1)];
          const uint32_t lo = v[i][e] & 0xFFFFu, hi = v[i][e] >> 16;
          const float s0 = (YT == CCQ_BF16 ? bf16_bits_to_f32(lo) : f16_bits_to_f32(lo)) + d[2 * (e & 1)] * f;
          const float s1 = (YT == CCQ_BF16 ? bf16_bits_to_f32(hi) : f16_bits_to_f32(hi)) + d[2 * (e & 1) + 1] * f;
          o[e] = YT == CCQ_BF16 ? bf16x2_bits(s0, s1) : f32_to_f16_bits(s0) | f32_to_f16_bits(s1) << 16;
        }
      }
      char* at = reinterpret_cast<char*>(y) + (row + n) * E;
      if (n + COLS <= N) {
        __builtin_memcpy(at, &o, 16);
      } else {
#pragma unroll
        for (int e = 0; e < COLS; ++e)
          if (n + e < N) {
            if constexpr (YT == CCQ_F32)
              reinterpret_cast<uint32_t*>(at)[e] = o[e];
            else
              reinterpret_cast<uint16_t*>(at)[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
          }
      }
    }
  }
};

// B rows of the 64 columns from n0 on, ranks c + 8 g .. of MFMA q
template <int WT, int YT>
__device__ __forceinline__ void lr_load_b(const LoraP& p, int adapter, int rank, int n0, int c, Raw<WT> (&w)[4]) {
  const int c16 = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int n = min(n0 + lr_col<YT>(q, c16), p.N - 1);  // columns past the end: not stored
    w[q] = lr_load<WT>(p.b, ((int64_t)adapter * p.N + n) * p.R, c + 8 * g, p.R);
  }
}

// acc[q] += B p for the 64 columns of w, one chunk of 32 ranks
template <int WT, int PARTS>
__device__ __forceinline__ void lr_expand_step(const Raw<WT> (&w)[4], const typename Half<WT>::vec (&pv)[PARTS],
                                               f32x4 (&acc)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
      acc[q] = lr_mfma(__builtin_bit_cast(typename Half<WT>::vec, w[q]), pv[i], acc[q]);
}

template <int YT>
__device__ __forceinline__ void lr_store(const LoraP& p, YBlock<YT>& y, int64_t row, int n0, int g,
                                         const f32x4 (&acc)[4], float f) {
  if constexpr (YT == CCQ_F32) {
    y.add_store(p.y, row, n0, g, p.N, acc, f);
  } else {  // both 16-bit types have one layout
    if (p.y_dtype == CCQ_BF16) {
      __builtin_bit_cast(YBlock<CCQ_BF16>, y).add_store(p.y, row, n0, g, p.N, acc, f);
    } else {
      __builtin_bit_cast(YBlock<CCQ_F16>, y).add_store(p.y, row, n0, g, p.N, acc, f);
    }
  }
}

// ------------------------------------------------------ one kernel (fused) --
// A workgroup: a tile of 16 tokens, ncols columns.  Its 8 waves split K, add
// their sums in LDS, and take blocks of 64 columns each; the first block's
// weights and y are loaded before the first product.
template <int XT, int WT, int YT, int RT>
__global__ __launch_bounds__(LR_THREADS) void lora_fused_kernel(const LoraP p) {
  using V = typename Half<WT>::vec;
  constexpr int PARTS = WT == CCQ_F16 ? 2 : YT == CCQ_F32 ? 3 : 2, RC = (RT + 1) / 2;
  __shared__ TileS<16> tl;
  __shared__ union {
    SortS<1> sort;
    f32x4 red[LR_WAVES][RT][64];
  } u;
  __shared__ __align__(16) float ps[16][32 * RC + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int tile = blockIdx.x % p.tiles, group = blockIdx.x / p.tiles;
  lr_find_tile<16, 1>(p, tile, tl, u.sort);
  const int adapter = tl.adapter;
  if (adapter < 0) return;
  const int rank = lr_rank(p, adapter);
  if (rank == 0) return;
  const float scale = p.scale != nullptr ? p.scale[adapter] : 1.f;
  const int own = tl.rows[c16], tok = own >= 0 ? own : tl.rows[0];  // padding: the first row again, not stored
  const int64_t xrow[1] = {(int64_t)tok * p.ldx}, yrow = (int64_t)tok * p.ldy;
  int64_t arow[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) arow[t] = ((int64_t)adapter * p.R + min(16 * t + c16, rank - 1)) * p.K;
  const int end = min((group + 1) * p.ncols, p.N);
  int n0 = group * p.ncols + 64 * wave;
  Raw<WT> w[RC][4];
  YBlock<YT> y;
  auto fetch = [&]() {
#pragma unroll
    for (int c = 0; c < RC; ++c) lr_load_b<WT, YT>(p, adapter, rank, n0, 32 * c, w[c]);
    y.load(p.y, yrow, n0, g, p.N);
  };
  if (n0 < end) fetch();
  f32x4 acc[1][RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int k0 = wave * p.kchunk;
  lr_shrink<XT, WT, 1, RT>(p, xrow, arow, k0, min(k0 + p.kchunk, p.K), acc);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; ++t) u.red[wave][t][lane] = acc[0][t];
  for (int i = threadIdx.x; i < 16 * (32 * RC - 16 * RT); i += LR_THREADS) ps[i & 15][16 * RT + (i >> 4)] = 0.f;
  __syncthreads();
  for (int t = wave; t < RT; t += LR_WAVES) {
    f32x4 s = u.red[0][t][lane];
#pragma unroll
    for (int k = 1; k < LR_WAVES; ++k) s += u.red[k][t][lane];
    // D: column (rank) lane & 15, row (token) 4 (lane >> 4) + i
#pragma unroll
    for (int i = 0; i < 4; ++i) ps[4 * g + i][16 * t + c16] = 16 * t + c16 < rank ? s[i] * scale : 0.f;
  }
  __syncthreads();
  if (n0 >= end) return;
  V pv[RC][PARTS];
  float down = 1.f;
  {
    float v[RC][8];
#pragma unroll
    for (int c = 0; c < RC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = ps[c16][32 * c + 8 * g + e];
    if constexpr (WT == CCQ_F16) {
      float m = 0.f;
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = isfinite(v[c][e]) ? fmaxf(m, fabsf(v[c][e])) : m;
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const int ex = lr_exponent(m);
      const float up = ldexpf(1.f, ex);
      down = ldexpf(1.f, -ex);
#pragma unroll
      for (int c = 0; c < RC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] *= up;
    }
#pragma unroll
    for (int c = 0; c < RC; ++c) lr_split<WT, PARTS>(v[c], pv[c]);
  }
  while (true) {
    f32x4 out[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) out[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      if (32 * c + 32 > rank) {  // the padding behind the rank may hold anything
#pragma unroll
        for (int q = 0; q < 4; ++q) lr_mask<WT>(w[c][q], rank - 32 * c - 8 * g);
      }
      lr_expand_step<WT, PARTS>(w[c], pv[c], out);
    }
    if (own >= 0) lr_store<YT>(p, y, yrow, n0, g, out, down);
    n0 += 64 * LR_WAVES;
    if (n0 >= end) break;
    fetch();
  }
}

// ------------------------------------------------------------ two kernels --
// A tile's 16 MT tokens, RT * 16 ranks from 16 RT blockIdx.z on, K range of
// one split, an eighth of it per wave.
template <int XT, int WT, int MT, int RT>
__global__ __launch_bounds__(LR_THREADS) void lora_shrink_kernel(const LoraP p) {
  constexpr int TM = 16 * MT, CH = MT == 1 ? 1 : LR_SELF / LR_THREADS;
  constexpr int PASS = MT * RT <= 8 ? MT : 8 / RT;  // row blocks whose sums are in LDS at once
  __shared__ TileS<TM> tl;
  __shared__ union {
    SortS<CH> sort;
    f32x4 red[LR_WAVES][PASS][RT][64];
  } u;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % p.S, tile = blockIdx.x / p.S;
  if (p.meta != nullptr) {
    lr_read_tile<TM>(p, tile, tl);
  } else {
    lr_find_tile<TM, CH>(p, tile, tl, u.sort);
    if (split == 0 && blockIdx.z == 0) {  // for the second kernel
      if (threadIdx.x < TM) p.tile_rows[(int64_t)tile * TM + threadIdx.x] = tl.rows[threadIdx.x];
      if (threadIdx.x == 0) p.tile_adapter[tile] = tl.adapter;
    }
  }
  const int adapter = tl.adapter;
  if (adapter < 0) return;
  const int rank = lr_rank(p, adapter), r0 = blockIdx.z * RT * 16;
  if (r0 >= rank) return;
  int64_t xrow[MT], arow[RT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int own = tl.rows[16 * m + c16];
    xrow[m] = (int64_t)(own >= 0 ? own : tl.rows[0]) * p.ldx;  // padding: the first row again, not stored
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) arow[t] = ((int64_t)adapter * p.R + min(r0 + 16 * t + c16, rank - 1)) * p.K;
  f32x4 acc[MT][RT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int kw = (p.kchunk / 32 + LR_WAVES - 1) / LR_WAVES * 32;  // per wave
  const int ks = split * p.kchunk, ke = min(ks + p.kchunk, p.K), k0 = ks + wave * kw;
  lr_shrink<XT, WT, MT, RT>(p, xrow, arow, k0, min(k0 + kw, ke), acc);
#pragma unroll
  for (int m0 = 0; m0 < MT; m0 += PASS) {
    __syncthreads();
#pragma unroll
    for (int m = 0; m < PASS; ++m)
#pragma unroll
      for (int t = 0; t < RT; ++t) u.red[wave][m][t][lane] = acc[m0 + m][t];
    __syncthreads();
    for (int i = wave; i < PASS * RT; i += LR_WAVES) {
      const int m = i / RT, t = i - m * RT;
      if (r0 + 16 * t >= rank) continue;  // the workspace's rows end with the last used 16 ranks
      f32x4 s = u.red[0][m][t][lane];
#pragma unroll
      for (int k = 1; k < LR_WAVES; ++k) s += u.red[k][m][t][lane];
      const int r = r0 + 16 * t + c16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // D: column (rank) lane & 15, row (token) 4 (lane >> 4) + e
        const int id = tl.rows[16 * (m0 + m) + 4 * g + e];
        if (id >= 0) p.p[((int64_t)split * p.T + id) * p.Rp + r] = r < rank ? s[e] : 0.f;
      }
    }
  }
}

// A tile's 16 MT tokens, ncols columns: p summed over the splits, scaled and
// in parts in LDS; the waves take blocks of 64 columns.
template <int WT, int YT, int MT>
__global__ __launch_bounds__(LR_THREADS) void lora_expand_kernel(const LoraP p) {
  using V = typename Half<WT>::vec;
  constexpr int PARTS = WT == CCQ_F16 ? 2 : YT == CCQ_F32 ? 3 : 2, TM = 16 * MT;
  __shared__ TileS<TM> tl;
  __shared__ float downs[TM];
  extern __shared__ __align__(16) uint16_t parts[];  // [PARTS][TM][ld]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int tile = blockIdx.x % p.tiles, group = blockIdx.x / p.tiles;
  lr_read_tile<TM>(p, tile, tl);
  const int adapter = tl.adapter;
  if (adapter < 0) return;
  const int rank = lr_rank(p, adapter);
  if (rank == 0) return;
  const float scale = p.scale != nullptr ? p.scale[adapter] : 1.f;
  const int rc = (rank + 31) / 32, r16 = (rank + 15) & ~15, ld = 32 * rc + 8;
  {  // 8 threads a row, each every eighth piece of 8 ranks
    const int row = threadIdx.x >> 3, j = threadIdx.x & 7;
    const int id = row < TM ? tl.rows[row] : -1;
    if (row < TM) {
      float v[LR_MAX_R / 64][8];
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < LR_MAX_R / 64; ++i) {
        const int r = 64 * i + 8 * j;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        if (id >= 0 && r < r16) {
          for (int s = 0; s < p.S; ++s) {
            float o[8];
            __builtin_memcpy(o, p.p + ((int64_t)s * p.T + id) * p.Rp + r, 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += o[e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[i][e] = r + e < rank ? v[i][e] * scale : 0.f;
            m = isfinite(v[i][e]) ? fmaxf(m, fabsf(v[i][e])) : m;
          }
        }
      }
      float up = 1.f, down = 1.f;
      if constexpr (WT == CCQ_F16) {
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const int ex = lr_exponent(m);
        up = ldexpf(1.f, ex);
        down = ldexpf(1.f, -ex);
      }
      if (j == 0) downs[row] = down;
#pragma unroll
      for (int i = 0; i < LR_MAX_R / 64; ++i) {
        const int r = 64 * i + 8 * j;
        if (r < 32 * rc) {
          V pv[PARTS];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] *= up;
          lr_split<WT, PARTS>(v[i], pv);
#pragma unroll
          for (int k = 0; k < PARTS; ++k) *reinterpret_cast<V*>(parts + (k * TM + row) * ld + r) = pv[k];
        }
      }
    }
  }
  __syncthreads();
  int64_t yrow[MT];
  bool own[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int id = tl.rows[16 * m + c16];
    own[m] = id >= 0;
    yrow[m] = (int64_t)(id >= 0 ? id : tl.rows[0]) * p.ldy;
  }
  const int end = min((group + 1) * p.ncols, p.N);
  for (int n0 = group * p.ncols + 64 * wave; n0 < end; n0 += 64 * LR_WAVES) {
    YBlock<YT> y[MT];
    f32x4 acc[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      y[m].load(p.y, yrow[m], n0, g, p.N);
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[m][q] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int c = 0; c < rc; ++c) {
      Raw<WT> w[4];
      lr_load_b<WT, YT>(p, adapter, rank, n0, 32 * c, w);
      if (32 * c + 32 > rank) {  // the padding behind the rank may hold anything
#pragma unroll
        for (int q = 0; q < 4; ++q) lr_mask<WT>(w[q], rank - 32 * c - 8 * g);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        V pv[PARTS];
#pragma unroll
        for (int k = 0; k < PARTS; ++k)
          pv[k] = *reinterpret_cast<const V*>(parts + (k * TM + 16 * m + c16) * ld + 32 * c + 8 * g);
        lr_expand_step<WT, PARTS>(w, pv, acc[m]);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (own[m]) lr_store<YT>(p, y[m], yrow[m], n0, g, acc[m], downs[16 * m + c16]);
  }
}

size_t a256l(size_t b) { return (b + 255) & ~(size_t)255; }

struct LoraPlan {
  bool fused, align;
  int64_t tm, tiles, S, kchunk, Rp, ncols;
  size_t off_rows, off_tile, off_meta, off_counts, off_align, off_p, total;
};

constexpr int64_t LR_FUSED_BYTES = 512 << 10;  // of one adapter's A

LoraPlan lora_plan(int64_t T, const ccq_lora_adapters* ad, bool one_type) {
  LoraPlan L = {};
  const int64_t K = ad->in_features, N = ad->out_features, R = ad->rank_max;
  L.Rp = cdiv(R, 16) * 16;
  L.fused = one_type && T <= LR_THREADS && R <= 128 && L.Rp * K * 2 <= LR_FUSED_BYTES;
  L.align = T > LR_SELF;
  L.tm = T <= LR_THREADS ? 16 : 64;
  L.tiles = ccq_moe_align_max_tiles(T, ad->num_adapters, L.tm);
  // 8 waves x 64 columns for a workgroup, or a multiple where that still gives two workgroups per CU
  const int64_t likely = L.tm == 16 ? L.tiles : cdiv(T, L.tm);
  int64_t groups = cdiv(N, 512);
  const int64_t want = cdiv(512, likely);
  if (groups > want) groups = want;
  L.ncols = cdiv(cdiv(N, groups), 512) * 512;
  if (L.fused) {
    L.S = 1;
    L.kchunk = cdiv(cdiv(K, 32), LR_WAVES) * 32;
    return L;
  }
  int64_t S = cdiv(512, likely);
  const int64_t most = cdiv(K, LR_WAVES * 64);
  S = S < most ? S : most;
  S = S < 8 ? S : 8;
  L.kchunk = cdiv(cdiv(K, S), 32) * 32;
  L.S = cdiv(K, L.kchunk);
  size_t o = 0;
  L.off_rows = o;
  o += a256l((size_t)L.tiles * L.tm * 4);
  L.off_tile = o;
  o += a256l((size_t)L.tiles * 4);
  L.off_meta = o;
  o += 256;
  L.off_counts = o;
  if (L.align) o += a256l((size_t)ad->num_adapters * 4);
  L.off_align = o;
  if (L.align) o += a256l(align_scratch_bytes(T, ad->num_adapters));
  L.off_p = o;
  o += a256l((size_t)L.S * T * L.Rp * 4);
  L.total = o;
  return L;
}

int check_adapters(const ccq_lora_adapters* ad, const char* name) {
  CCQ_REQUIRE(ad != nullptr, "%s: null adapter descriptor", name);
  CCQ_REQUIRE(ad->dtype == CCQ_F16 || ad->dtype == CCQ_BF16, "%s: adapters must be f16 or bf16", name);
  CCQ_REQUIRE(ad->num_adapters >= 1 && ad->num_adapters <= LR_MAX_L, "%s: num_adapters=%lld outside [1, %d]", name,
              (long long)ad->num_adapters, LR_MAX_L);
  CCQ_REQUIRE(ad->rank_max >= 1 && ad->rank_max <= LR_MAX_R, "%s: rank_max=%lld outside [1, %d]", name,
              (long long)ad->rank_max, LR_MAX_R);
  CCQ_REQUIRE(ad->in_features >= 1 && ad->in_features <= (1 << 20) && ad->out_features >= 1 &&
                  ad->out_features <= (1 << 20),
              "%s: in_features=%lld and out_features=%lld must be in [1, 2^20]", name, (long long)ad->in_features,
              (long long)ad->out_features);
  return 0;
}

template <int XT, int WT, int YT>
void fused_launch(const LoraP& p, int64_t groups, hipStream_t st) {
  const int rt = (int)cdiv(p.R, 16);
  const dim3 grid((unsigned)(p.tiles * groups)), block(LR_THREADS);
  if (rt <= 1)
    launch((lora_fused_kernel<XT, WT, YT, 1>), grid, block, 0, st, p);
  else if (rt <= 2)
    launch((lora_fused_kernel<XT, WT, YT, 2>), grid, block, 0, st, p);
  else if (rt <= 4)
    launch((lora_fused_kernel<XT, WT, YT, 4>), grid, block, 0, st, p);
  else
    launch((lora_fused_kernel<XT, WT, YT, 8>), grid, block, 0, st, p);
}

template <int XT, int WT>
void fused_dispatch(const LoraP& p, int64_t groups, hipStream_t st) {
  if (p.y_dtype == CCQ_F32)
    fused_launch<XT, WT, CCQ_F32>(p, groups, st);
  else  // both 16-bit types
    fused_launch<XT, WT, CCQ_BF16>(p, groups, st);
}

template <int XT, int WT, int MT>
void shrink_launch(const LoraP& p, hipStream_t st) {
  const int rt = (int)cdiv(p.R, 16);
  const dim3 block(LR_THREADS);
  const unsigned x = (unsigned)(p.tiles * p.S);
  if (rt <= 1)
    launch((lora_shrink_kernel<XT, WT, MT, 1>), dim3(x), block, 0, st, p);
  else if (rt <= 2)
    launch((lora_shrink_kernel<XT, WT, MT, 2>), dim3(x), block, 0, st, p);
  else if (rt <= 4)
    launch((lora_shrink_kernel<XT, WT, MT, 4>), dim3(x), block, 0, st, p);
  else
    launch((lora_shrink_kernel<XT, WT, MT, 8>), dim3(x, 1, (unsigned)cdiv(rt, 8)), block, 0, st, p);
}

template <int WT, int MT>
void expand_launch(const LoraP& p, int64_t groups, hipStream_t st) {
  const dim3 grid((unsigned)(p.tiles * groups)), block(LR_THREADS);
  const size_t ld = (size_t)cdiv(p.R, 32) * 32 + 8, part = ld * 16 * MT * 2;
  if (p.y_dtype == CCQ_F32)
    launch((lora_expand_kernel<WT, CCQ_F32, MT>), grid, block, part * (WT == CCQ_BF16 ? 3 : 2), st, p);
  else
    launch((lora_expand_kernel<WT, CCQ_BF16, MT>), grid, block, part * 2, st, p);
}

template <int WT, int MT>
int two_launches(const LoraP& p, int x_dtype, int64_t groups, hipStream_t st) {
  if (x_dtype == CCQ_BF16)
    shrink_launch<CCQ_BF16, WT, MT>(p, st);
  else if (x_dtype == CCQ_F16)
    shrink_launch<CCQ_F16, WT, MT>(p, st);
  else
    shrink_launch<CCQ_F32, WT, MT>(p, st);
  if (int rc = launch_status("ccq_lora_add (shrink)")) return rc;
  expand_launch<WT, MT>(p, groups, st);
  return launch_status("ccq_lora_add (expand)");
}

bool lora_float_code(int dt) { return dt == CCQ_F32 || dt == CCQ_F16 || dt == CCQ_BF16; }
bool lora_one_type(int x_dtype, const ccq_lora_adapters* ad) { return x_dtype == CCQ_F32 || x_dtype == ad->dtype; }

}  // namespace

}  // namespace ccq

using namespace ccq;

extern "C" size_t ccq_lora_workspace_size(int64_t T, int x_dtype, const ccq_lora_adapters* ad) {
  if (T <= 0 || T > 65536 || !lora_float_code(x_dtype) || check_adapters(ad, "ccq_lora_workspace_size")) return 0;
  return lora_plan(T, ad, lora_one_type(x_dtype, ad)).total;
}

extern "C" int ccq_lora_add(const void* x, int x_dtype, int64_t ldx, const int64_t* index, void* y, int y_dtype,
                            int64_t ldy, int64_t T, const ccq_lora_adapters* ad, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (int rc = check_adapters(ad, "ccq_lora_add")) return rc;
  CCQ_REQUIRE(T >= 0 && T <= 65536, "ccq_lora_add: T=%lld outside [0, 65536]", (long long)T);
  CCQ_REQUIRE(lora_float_code(x_dtype), "ccq_lora_add: bad x_dtype");
  CCQ_REQUIRE(lora_float_code(y_dtype), "ccq_lora_add: bad y_dtype");
  CCQ_REQUIRE(ldx >= ad->in_features && ldy >= ad->out_features, "ccq_lora_add: a row stride below the row's length");
  if (T == 0) return 0;
  CCQ_REQUIRE(x && index && y && ad->a && ad->b, "ccq_lora_add: null pointer");
  CCQ_REQUIRE(aligned(x, x_dtype == CCQ_F32 ? 4 : 2) && aligned(y, y_dtype == CCQ_F32 ? 4 : 2) && aligned(index, 8) &&
                  aligned(ad->a, 2) && aligned(ad->b, 2) && aligned(ad->scale, 4) && aligned(ad->rank, 4),
              "ccq_lora_add: a pointer is not aligned to its elements");
  const LoraPlan L = lora_plan(T, ad, lora_one_type(x_dtype, ad));
  CCQ_REQUIRE(L.total == 0 || (workspace && workspace_bytes >= L.total && aligned(workspace, 256)),
              "ccq_lora_add: workspace of %zu bytes (256-byte aligned) needed, %zu given", L.total, workspace_bytes);
  hipStream_t st = as_stream(stream);
  char* ws = (char*)workspace;
  const int64_t groups = cdiv(ad->out_features, L.ncols);
  LoraP p = {};
  p.x = x;
  p.y = y;
  p.index = index;
  p.a = ad->a;
  p.b = ad->b;
  p.scale = ad->scale;
  p.rank = ad->rank;
  p.ldx = ldx;
  p.ldy = ldy;
  p.T = (int)T;
  p.L = (int)ad->num_adapters;
  p.R = (int)ad->rank_max;
  p.Rp = (int)L.Rp;
  p.K = (int)ad->in_features;
  p.N = (int)ad->out_features;
  p.S = (int)L.S;
  p.kchunk = (int)L.kchunk;
  p.tiles = (int)L.tiles;
  p.ncols = (int)L.ncols;
  p.y_dtype = y_dtype;
  if (L.fused) {
    if (ad->dtype == CCQ_BF16) {
      if (x_dtype == CCQ_F32)
        fused_dispatch<CCQ_F32, CCQ_BF16>(p, groups, st);
      else
        fused_dispatch<CCQ_BF16, CCQ_BF16>(p, groups, st);
    } else {
      if (x_dtype == CCQ_F32)
        fused_dispatch<CCQ_F32, CCQ_F16>(p, groups, st);
      else
        fused_dispatch<CCQ_F16, CCQ_F16>(p, groups, st);
    }
    return launch_status("ccq_lora_add");
  }
  p.tile_rows = (int32_t*)(ws + L.off_rows);
  p.tile_adapter = (int32_t*)(ws + L.off_tile);
  p.p = (float*)(ws + L.off_p);
  if (L.align) {
    p.meta = (const int32_t*)(ws + L.off_meta);
    const int rc = launch_align(index, T, p.L, L.tm, p.tile_rows, p.tile_adapter, (int32_t*)(ws + L.off_meta),
                                (int32_t*)(ws + L.off_counts), st, ws + L.off_align, align_scratch_bytes(T, p.L));
    if (rc) return rc;
  }
  if (ad->dtype == CCQ_BF16)
    return L.tm == 16 ? two_launches<CCQ_BF16, 1>(p, x_dtype, groups, st)
                      : two_launches<CCQ_BF16, 4>(p, x_dtype, groups, st);
  return L.tm == 16 ? two_launches<CCQ_F16, 1>(p, x_dtype, groups, st)
                    : two_launches<CCQ_F16, 4>(p, x_dtype, groups, st);
}
