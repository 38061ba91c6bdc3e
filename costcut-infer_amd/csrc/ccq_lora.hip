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
//
// p stays float32 between the products.  The second one takes it in parts of
// the weights' type (lr_split) whose sum is p to 16 bits or more, so that y's
// own rounding is the only one that shows; sums are float32 everywhere.
//
// What bounds it: prompts, y read and written once and x read once (T=2048
// K=4096 N=14336 R=16: 134 MB, 34 us, 4.1 TB/s); a batch of few tokens, the
// chain index -> tile -> A, x, B, y -> LDS -> store, 6 to 9 us in one kernel,
// 11 to 16 in two.
#include "ccq_common.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace ccq {

namespace {

constexpr int LR_THREADS = 512, LR_WAVES = 8;
constexpr int LE_THREADS = 256;  // of the expand kernel
constexpr int LR_MAX_R = 256;
constexpr int LR_MAX_L = 1024;
constexpr int LR_SELF = 4096;   // most tokens that workgroups sort themselves: 8 a thread (T=4096 K=N=2048 R=16 21.8 us,
                                // behind the schedule's own launch 26.0; T=1100 15.6 and 18.4)

struct LoraP {
  const void* x;
  void* y;
  const int64_t* index;
  const void* a;
  const void* b;
  const float* scale;
  const int32_t* rank;
  int32_t* tile_rows;           // [tiles][TM], -1: padding
  int32_t* tile_adapter;        // [tiles], of ccq_moe_align's schedule
  int4* tile_info;              // [tiles], for the second kernel: adapter (-1: no such tile), rank, bits of the scale, splits
  const int32_t* meta;          // tiles of ccq_moe_align's schedule; null: workgroups sort
  float* p;                     // [S][T][Rp]
  int64_t ldx, ldy;
  int64_t last_x, last_a, last_b;  // where the last 8 values of x, a and b begin
  int T, L, R, Rp, K, N;
  int S, kchunk;                // splits of K, K per split (a multiple of 32)
  int few, S_few, kchunk_few;   // those of the 64-token shrink for up to `few` tiles
  int tiles, ncols;             // tiles of the grid, columns per workgroup
  int y_dtype;
};

template <int DT>
struct Half;
template <>
struct Half<CCQ_BF16> {
  using vec = bf16x8;
  using quad = __bf16 __attribute__((ext_vector_type(4)));
};
template <>
struct Half<CCQ_F16> {
  using vec = f16x8;
  using quad = _Float16 __attribute__((ext_vector_type(4)));
};

__device__ __forceinline__ f32x4 lr_mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 lr_mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 8 values from element i on of a buffer whose last 8 begin at `last`, as
// loaded: one load at any element alignment, of those last 8 where i is past
// them.  lr_fix then moves the values to their places and clears those from n
// on; until then they may be other rows' values.
template <int DT>
struct Raw {
  u32x4 v[DT == CCQ_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw<DT> lr_load_whole(const void* base, int64_t i) {
  constexpr int E = DT == CCQ_F32 ? 4 : 2;
  Raw<DT> r;
  __builtin_memcpy(&r, reinterpret_cast<const char*>(base) + i * E, 8 * E);
  return r;
}
template <int DT>
__device__ __forceinline__ Raw<DT> lr_load(const void* base, int64_t i, int64_t last) {
  return lr_load_whole<DT>(base, i < last ? i : last);
}
template <int DT>
__device__ __forceinline__ void lr_fix(Raw<DT>& r, int64_t i, int64_t last, int n) {
  constexpr int W = DT == CCQ_F32 ? 8 : 4;
  const int s = i <= last ? 0 : i - last < 8 ? (int)(i - last) : 8;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
  const int words = DT == CCQ_F32 ? s : s >> 1;
#pragma unroll
  for (int step = W / 2; step >= 1; step >>= 1)
#pragma unroll
    for (int e = 0; e < W; ++e) w[e] = words & step ? (e + step < W ? w[e + step] : 0u) : w[e];
  if constexpr (DT != CCQ_F32) {
#pragma unroll
    for (int e = 0; e < W; ++e) w[e] = s & 1 ? w[e] >> 16 | (e + 1 < W ? w[e + 1] << 16 : 0u) : w[e];
  }
  if (s >= 8) n = 0;
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
// such tile) and token ids.  Wave w holds tokens 64 (w CH + c) + lane;
// pick(number of tiles) is the tile.
template <int TM>
struct TileS {
  int adapter, first;           // first: the tile's place among its adapter's
  int rows[TM];
};
struct SortS {
  int count[LR_MAX_L];
  int sum[LR_WAVES];
};

template <int TM, int CH, class Pick>
__device__ void lr_find_tile(const LoraP& p, Pick pick, TileS<TM>& t, SortS& s) {
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
  int sum = wave_scan(n0 + n1);
  if (lane == 63) s.sum[wave] = sum;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < LR_WAVES - 1; ++w) sum += w < wave ? s.sum[w] : 0;
  int total = 0;
#pragma unroll
  for (int w = 0; w < LR_WAVES; ++w) total += s.sum[w];
  const int tile = pick(total);
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
#pragma unroll
  for (int w = 0; w < LR_WAVES - 1; ++w) pos += w < wave ? s.sum[w] : 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint64_t m = __ballot(key[c] == adapter);
    const int at = pos + __popcll(m & ((1ull << lane) - 1));
    if (key[c] == adapter && at >= 0 && at < TM) t.rows[at] = 64 * (wave * CH + c) + lane;
    pos += __popcll(m);
  }
  __syncthreads();
}

// The same for up to 64 tokens and tiles of 16, by each wave for itself: lane t
// holds token t.  Lane r < 16 returns the tile's row r (-1: padding).
__device__ __forceinline__ int lr_find_tile_wave(const LoraP& p, int tile, int& adapter) {
  const int lane = threadIdx.x & 63;
  const int64_t i = lane < p.T ? p.index[lane] : -1;
  const int key = i >= 0 && i < p.L ? (int)i : -1;
  uint64_t same = __ballot(key >= 0);  // the tokens of this lane's adapter
  for (int b = 0; (p.L - 1) >> b; ++b) {
    const uint64_t m = __ballot((key >> b) & 1);
    same &= (key >> b) & 1 ? m : ~m;
  }
  const bool head = key >= 0 && (same & ((1ull << lane) - 1)) == 0;
  int n = head ? (__popcll(same) + 15) >> 4 : 0;  // tiles of this lane's adapter
  int start;
  if (__ballot(n > 1) == 0) {
    start = __popcll(__ballot(head) & ((1ull << lane) - 1));
  } else {
    start = wave_scan(n) - n;
  }
  const uint64_t hit = __ballot(head && tile >= start && tile < start + n);
  adapter = -1;
  if (hit == 0) return -1;
  const int l = __builtin_ctzll(hit);
  adapter = __builtin_amdgcn_readlane(key, l);
  const int first = 16 * (tile - __builtin_amdgcn_readlane(start, l));
  const uint64_t group = __ballot(key == adapter);
  // token t of the adapter's rank j goes to lane j - first, the others to lane 63
  const int j = __popcll(group & ((1ull << lane) - 1)) - first;
  const bool in = key == adapter && j >= 0 && j < 16;
  const int got = __builtin_amdgcn_ds_permute(4 * (in ? j : 63), lane);
  return lane < min(16, __popcll(group) - first) ? got : -1;
}

// the same from a finished schedule
template <int TM>
__device__ void lr_read_tile(const LoraP& p, int tile, TileS<TM>& t) {
  const bool none = p.meta != nullptr && tile >= p.meta[0];
  if (threadIdx.x < TM) t.rows[threadIdx.x] = none ? -1 : p.tile_rows[(int64_t)tile * TM + threadIdx.x];
  if (threadIdx.x == 0) t.adapter = none ? -1 : p.tile_adapter[tile];
  __syncthreads();
}

// what the second kernel needs of a tile in one load
__device__ __forceinline__ void lr_write_info(const LoraP& p, int tile, int adapter, int rank, int splits) {
  if (threadIdx.x == 0)
    p.tile_info[tile] = make_int4(rank > 0 ? adapter : -1, rank,
                                  __float_as_int(adapter >= 0 && p.scale != nullptr ? p.scale[adapter] : 1.f), splits);
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

// Tile and split of a workgroup of the shrink kernels: tiles dealt to the XCDs
// one by one, all splits of one together.  (Runs of tiles on an XCD would share
// A in its L2, but the tiles that the grid has beyond the real ones then idle
// whole XCDs: T=64 K=14336 R=128, 16 tiles of at most 20, 24 us against 15.)
__device__ __forceinline__ int lr_tile_of(const LoraP& p, int& split) {
  const int local = blockIdx.x >> 3, t = local / p.S;
  split = local - t * p.S;
  return t * 8 + (blockIdx.x & 7);
}

// U k-steps whose loads are in flight together, as often as they fit, then half as many
template <int XT, int WT, int MT, int RT, int U>
__device__ __forceinline__ void lr_steps(const LoraP& p, const int64_t (&xrow)[MT], const int64_t (&arow)[RT], int& k,
                                         int k1, f32x4 (&acc)[MT][RT]) {
  const int g = (threadIdx.x >> 4) & 3;
  for (; k + 32 * U <= k1; k += 32 * U) {
    Raw<XT> xr[U][MT];
    Raw<WT> ar[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int m = 0; m < MT; ++m) xr[u][m] = lr_load_whole<XT>(p.x, xrow[m] + k + 32 * u + 8 * g);
#pragma unroll
      for (int t = 0; t < RT; ++t) ar[u][t] = lr_load_whole<WT>(p.a, arow[t] + k + 32 * u + 8 * g);
    }
    __builtin_amdgcn_sched_barrier(0);  // all of them before the first product
#pragma unroll
    for (int u = 0; u < U; ++u) lr_multiply<XT, WT, MT, RT>(xr[u], ar[u], acc);
  }
  if constexpr (U > 1) lr_steps<XT, WT, MT, RT, U / 2>(p, xrow, arow, k, k1, acc);
}

template <int XT, int WT, int MT, int RT, int U>
__device__ __forceinline__ void lr_shrink(const LoraP& p, const int64_t (&xrow)[MT], const int64_t (&arow)[RT], int k0,
                                          int k1, f32x4 (&acc)[MT][RT]) {
  const int g = (threadIdx.x >> 4) & 3;
  int k = k0;
  lr_steps<XT, WT, MT, RT, U>(p, xrow, arow, k, k1, acc);
  if (k < k1) {  // the last, partial step of K
    const int kk = k + 8 * g;
    Raw<XT> xr[MT];
    Raw<WT> ar[RT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m] = lr_load<XT>(p.x, xrow[m] + kk, p.last_x);
#pragma unroll
    for (int t = 0; t < RT; ++t) ar[t] = lr_load<WT>(p.a, arow[t] + kk, p.last_a);
#pragma unroll
    for (int m = 0; m < MT; ++m) lr_fix<XT>(xr[m], xrow[m] + kk, p.last_x, p.K - kk);
#pragma unroll
    for (int t = 0; t < RT; ++t) lr_fix<WT>(ar[t], arow[t] + kk, p.last_a, p.K - kk);
    lr_multiply<XT, WT, MT, RT>(xr, ar, acc);
  }
}

// Stages of whole 128-byte lines of x's rows, D - 1 of them loaded
// ahead of the products: for the 64-token tiles of rows that are not aligned,
// whose waves walk far in K.
template <int XT, int WT, int MT, int RT, int D>
__device__ __forceinline__ void lr_shrink_ring(const LoraP& p, const int64_t (&xrow)[MT], const int64_t (&arow)[RT],
                                               int k0, int k1, f32x4 (&acc)[MT][RT]) {
  const int g = (threadIdx.x >> 4) & 3;
  constexpr int SU = XT == CCQ_F32 ? 1 : 2, SK = 32 * SU;
  const int n = k1 > k0 ? (k1 - k0) / SK : 0;
  Raw<XT> xr[D][SU][MT];
  Raw<WT> ar[D][SU][RT];
  auto load = [&](int s, int d) {
    const int k = k0 + SK * s + 8 * g;
#pragma unroll
    for (int u = 0; u < SU; ++u) {
#pragma unroll
      for (int m = 0; m < MT; ++m) xr[d][u][m] = lr_load_whole<XT>(p.x, xrow[m] + k + 32 * u);
#pragma unroll
      for (int t = 0; t < RT; ++t) ar[d][u][t] = lr_load_whole<WT>(p.a, arow[t] + k + 32 * u);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (n > 0) {
#pragma unroll
    for (int d = 0; d < D - 1; ++d) load(min(d, n - 1), d);  // past the range: its last stage again, not multiplied
    for (int s = 0; s < n; s += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        load(min(s + d + D - 1, n - 1), (d + D - 1) % D);
        if (s + d < n) {
#pragma unroll
          for (int u = 0; u < SU; ++u) lr_multiply<XT, WT, MT, RT>(xr[d][u], ar[d][u], acc);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  lr_shrink<XT, WT, MT, RT, 1>(p, xrow, arow, k0 + SK * n, k1, acc);  // what is left: less than a stage
}

// ---------------------------------------------------------------- expand --
// p in parts of the weights' type, most significant first, whose sum is p to
// 16 (two parts of bf16), 24 (three) or 22 bits of the row's largest (two of
// f16, the row scaled by a power of two into its range).  Parts in bf16 end at
// 2^-133, so a p below 2^-105 keeps fewer bits of three; they are taken of p / 4
// (LR_DOWN), since a p of 2^128 (1 - 2^-9) and more rounds to infinity in bf16.
template <int WT>
constexpr float LR_DOWN = WT == CCQ_BF16 ? 4.f : 1.f;
template <int WT, int PARTS, int N, class V>
__device__ __forceinline__ void lr_split(const float (&v)[N], V (&out)[PARTS]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
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

// the value whose parts lie `stride` values apart
template <int WT, int PARTS>
__device__ __forceinline__ float lr_join(const uint16_t* parts, int stride) {
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < PARTS; ++i)
    v += WT == CCQ_BF16 ? bf16_bits_to_f32(parts[i * stride]) : f16_bits_to_f32(parts[i * stride]);
  return v;
}

// k such that 2^k brings a row whose largest finite |p| is m into [2^13, 2^14],
// from -114 (m near 2^128) on, up to what lr_pow2 holds of 2^k and 2^-k: below
// 2^-112 m stays smaller (2^-126 becomes 1), and the parts, which end at 2^-24,
// still hold 22 bits of it.
__device__ __forceinline__ int lr_exponent(float m) {
  return m > 0.f ? min(14 - __builtin_amdgcn_frexp_expf(m), 126) : 0;
}
__device__ __forceinline__ float lr_pow2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }

// 16 bytes of a row of y from column n on (at any element alignment).  A piece
// across the row's end is not loaded, and added to in place value by value.
// YT: float32, or either 16-bit type (they differ in the sums alone).
template <int YT>
struct YPiece {
  static constexpr int COLS = YT == CCQ_F32 ? 4 : 8;
  u32x4 v;
  __device__ __forceinline__ void load(const void* y, int64_t row, int n, int N) {
    constexpr int E = YT == CCQ_F32 ? 4 : 2;
    v = u32x4{0, 0, 0, 0};
    if (n + COLS <= N) __builtin_memcpy(&v, reinterpret_cast<const char*>(y) + (row + n) * E, 16);
  }
  // the piece with d added; DT: y's type
  template <int DT>
  __device__ __forceinline__ u32x4 sum(const float (&d)[COLS]) const {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == CCQ_F32)
        o[e] = __float_as_uint(__uint_as_float(v[e]) + d[e]);
      else if constexpr (DT == CCQ_BF16)
        o[e] = bf16x2_bits(bf16_bits_to_f32(v[e] & 0xFFFFu) + d[2 * e], bf16_bits_to_f32(v[e] >> 16) + d[2 * e + 1]);
      else
        o[e] = f32_to_f16_bits(f16_bits_to_f32(v[e] & 0xFFFFu) + d[2 * e]) |
               f32_to_f16_bits(f16_bits_to_f32(v[e] >> 16) + d[2 * e + 1]) << 16;
    }
    return o;
  }
  __device__ __forceinline__ void add_store(void* y, int y_dtype, int64_t row, int n, int N, const float (&d)[COLS]) {
    constexpr int E = YT == CCQ_F32 ? 4 : 2;
    char* at = reinterpret_cast<char*>(y) + (row + n) * E;
    if (n + COLS <= N) {
      u32x4 o;
      if constexpr (YT == CCQ_F32)
        o = sum<CCQ_F32>(d);
      else if (y_dtype == CCQ_BF16)
        o = sum<CCQ_BF16>(d);
      else
        o = sum<CCQ_F16>(d);
      __builtin_memcpy(at, &o, 16);
    } else {
#pragma unroll
      for (int e = 0; e < COLS; ++e)
        if (n + e < N) {
          if constexpr (YT == CCQ_F32) {
            reinterpret_cast<float*>(at)[e] += d[e];
          } else {
            uint16_t* h = reinterpret_cast<uint16_t*>(at) + e;
            *h = (uint16_t)(y_dtype == CCQ_BF16 ? bf16x2_bits(bf16_bits_to_f32(*h) + d[e], 0.f)
                                                : f32_to_f16_bits(f16_bits_to_f32(*h) + d[e]));
          }
        }
    }
  }
};

// Column of D row m of MFMA q in a block of 64: a lane's quads join to 16-byte
// pieces of its token's row, four lanes to 64 contiguous bytes.
template <int YT>
__device__ __forceinline__ int lr_col(int q, int m) {
  return YT == CCQ_F32 ? 16 * q + m : 32 * (q >> 1) + 8 * (m >> 2) + 4 * (q & 1) + (m & 3);
}
// where piece i of lane group g begins, and its values among the lane's quads
template <int YT>
__device__ __forceinline__ int lr_piece_col(int i, int g) { return YT == CCQ_F32 ? 16 * i + 4 * g : 32 * i + 8 * g; }
// Lanes of one wave hand each other values through LDS: the hardware keeps a
// wave's LDS accesses in order, the fences keep the compiler from moving them
// across.  They emit no instruction.
__device__ __forceinline__ void lr_lane_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// An infinite weight times p's parts is NaN where these differ in sign or one
// is 0.  Where a column has such a weight, its sums that are NaN are formed anew
// from whole p(row, r): `sums` holds the wave's 64 columns from n0 on, a row of
// them for each of ROWS tokens.  (p joined from f16 parts is 0 below 2^-38 of
// its row's largest.)  The lane and the scan of b one by one: what is alive in
// the kernels' loops leaves few registers.  The check of the sums costs T=16
// K=4096 N=14336 R=16 0.2 of 8.4 us and T=4096 N=4096 R=128 0.1 of 71.7 a call;
// x that is NaN throughout, which scans b for nothing, takes 44 -> 154 us there
// with K=2048.
template <int WT, int ROWS, class F>
__device__ __forceinline__ void lr_whole_sums(const LoraP& p, int adapter, int rank, int n0, float (*sums)[64 + 4], F whole) {
  const int lane = lane_id_here();
  const uint16_t* b = reinterpret_cast<const uint16_t*>(p.b) + ((int64_t)adapter * p.N + min(n0 + lane, p.N - 1)) * p.R;
  bool inf = false;
#pragma unroll 1
  for (int r = 0; r < rank; ++r) inf |= (b[r] & 0x7FFF) == (WT == CCQ_BF16 ? 0x7F80 : 0x7C00);
  if (!inf) return;
#pragma unroll 1
  for (int i = 0; i < ROWS; ++i) {
    if (sums[i][lane] == sums[i][lane]) continue;
    float sum = 0.f;
#pragma unroll 1
    for (int r = 0; r < rank; ++r)
      sum = fmaf(whole(i, r), WT == CCQ_BF16 ? bf16_bits_to_f32(b[r]) : f16_bits_to_f32(b[r]), sum);
    sums[i][lane] = sum;
  }
}

// not a number if one of acc is none (or where their products leave the range)
__device__ __forceinline__ float lr_nan_of(const f32x4 (&acc)[4]) {
  float t = 0.f;
#pragma unroll
  for (int q = 0; q < 4; ++q) t = fmaf(acc[q][2], acc[q][3], fmaf(acc[q][0], acc[q][1], t));
  return t;
}

// (The branches between whole and ragged blocks and between the types stand once,
// around all pieces: a kernel of a few us pays for the code that it steps over.
// T=16 K=4096 N=14336 R=16 9.4 us on the GPU by branches in each piece, 9.2 so.)
template <int YT>
__device__ __forceinline__ void lr_store_pieces(const LoraP& p, YPiece<YT> (&y)[16 / YPiece<YT>::COLS], int64_t row,
                                                int n0, int g, const f32x4 (&acc)[4], float f) {
  constexpr int C = YPiece<YT>::COLS, E = YT == CCQ_F32 ? 4 : 2;
  float d[16 / C][C];
#pragma unroll
  for (int i = 0; i < 16; ++i) d[i / C][i % C] = acc[i / 4][i & 3] * f;
  if (__builtin_expect(n0 + 64 <= p.N, 1)) {
    char* at = reinterpret_cast<char*>(p.y) + (row + n0 + lr_piece_col<YT>(0, g)) * E;
    auto store = [&](auto dt) {
#pragma unroll
      for (int i = 0; i < 16 / C; ++i) {
        const u32x4 o = y[i].template sum<decltype(dt)::value>(d[i]);
        __builtin_memcpy(at + lr_piece_col<YT>(i, 0) * E, &o, 16);
      }
    };
    if constexpr (YT == CCQ_F32)
      store(std::integral_constant<int, CCQ_F32>{});
    else if (p.y_dtype == CCQ_BF16)
      store(std::integral_constant<int, CCQ_BF16>{});
    else
      store(std::integral_constant<int, CCQ_F16>{});
  } else {
#pragma unroll
    for (int i = 0; i < 16 / C; ++i) y[i].add_store(p.y, p.y_dtype, row, n0 + lr_piece_col<YT>(i, g), p.N, d[i]);
  }
}

// B rows of 64 columns from n0 on, ranks c + 8 g .. (columns past the end
// repeat the last one: not stored), and, in the last chunk, its part behind
// the rank cleared: the padding there may hold anything.  col(q): the column
// of this lane's row of MFMA q.
template <int WT, typename F>
__device__ __forceinline__ void lr_load_b(const LoraP& p, int adapter, int c, F col, Raw<WT> (&w)[4]) {
  const int r = c + 8 * ((threadIdx.x >> 4) & 3);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    w[q] = lr_load<WT>(p.b, ((int64_t)adapter * p.N + min(col(q), p.N - 1)) * p.R + r, p.last_b);
}
template <int WT, typename F>
__device__ __forceinline__ void lr_fix_b(const LoraP& p, int adapter, int rank, int c, F col, Raw<WT> (&w)[4]) {
  const int r = c + 8 * ((threadIdx.x >> 4) & 3);
  if (c + 32 <= rank) return;
  if (p.R % 8 == 0) {  // whole pieces: the same mask for all rows
    uint32_t keep[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      keep[e] = (r + 2 * e < rank ? 0xFFFFu : 0u) | (r + 2 * e + 1 < rank ? 0xFFFF0000u : 0u);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[q].v[0][e] &= keep[e];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      lr_fix<WT>(w[q], ((int64_t)adapter * p.N + min(col(q), p.N - 1)) * p.R + r, p.last_b, rank - r);
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

// ------------------------------------------------------ one kernel (fused) --
// A workgroup: a tile of 16 tokens, ncols columns.  The lines (64 k) of x and A
// are dealt to its 8 waves, each copying its own into its part of LDS, D of
// them ahead, and multiplying them without a barrier: a load that takes 8 rows
// x 128 bytes reads 145 GB/s on a CU (131 KB by 8 waves, from L2), the
// operands' own 16 rows x 64 bytes 40 GB/s.  The sums meet in LDS; the waves
// then take blocks of 64 columns each, the first one's weights and y loaded
// before the first product.  Rows are aligned to 16 bytes here.  In a line the
// 16-byte piece i of row r lies at i ^ (r & 7), so that the operand reads of 8
// neighbouring lanes cover all banks.
template <int XT, int WT, int YT, int RT>
__global__ __launch_bounds__(LR_THREADS) void lora_fused_kernel(const LoraP p) {
  using V = typename Half<WT>::vec;
  constexpr int PARTS = WT == CCQ_F16 ? 2 : YT == CCQ_F32 ? 3 : 2, RC = (RT + 1) / 2;
  constexpr int E = XT == CCQ_F32 ? 4 : 2, XL = E / 2;  // lines of x for 64 k
  constexpr int BYTES = (XL + RT) * 2048, NI = BYTES / 1024, D = 18 * 1024 / BYTES;
  static_assert(D >= 2 && D <= 4 && D * BYTES >= RT * 1024);
  __shared__ TileS<16> tl;
  __shared__ __align__(16) union {
    SortS sort;
    char ring[LR_WAVES][D][BYTES];
    f32x4 red[LR_WAVES][RT][64];
  } u;
  __shared__ __align__(16) float ps[16][32 * RC + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
  // all workgroups of a tile on one XCD, whose L2 then holds its A
  const int t8 = (p.tiles + 7) & ~7, tile = blockIdx.x % t8, group = blockIdx.x / t8;
  if (tile >= p.tiles) return;
  int adapter, rows;  // lane r < 16: the tile's row r
  if (p.T <= 64) {
    rows = lr_find_tile_wave(p, tile, adapter);
  } else {
    lr_find_tile<16, 1>(p, [&](int) { return tile; }, tl, u.sort);
    adapter = tl.adapter;
    rows = tl.rows[c16];
  }
  adapter = __builtin_amdgcn_readfirstlane(adapter);
  if (adapter < 0) return;
  const int rank = __builtin_amdgcn_readfirstlane(lr_rank(p, adapter));
  if (rank == 0) return;
  const float scale = (p.scale != nullptr ? p.scale[adapter] : 1.f) / LR_DOWN<WT>;
  const int own = __shfl(rows, c16, 64), row0 = __shfl(rows, 0, 64);
  const int64_t yrow = (int64_t)(own >= 0 ? own : row0) * p.ldy;  // padding: the first row again, not stored

  const int end = min((group + 1) * p.ncols, p.N);
  int n0 = group * p.ncols + 64 * wave;
  auto col = [&](int q) { return n0 + lr_col<YT>(q, c16); };
  Raw<WT> w[RC][4];
  YPiece<YT> y[16 / YPiece<YT>::COLS];
  auto fetch = [&]() {
#pragma unroll
    for (int c = 0; c < RC; ++c) lr_load_b<WT>(p, adapter, 32 * c, col, w[c]);
#pragma unroll
    for (int i = 0; i < 16 / YPiece<YT>::COLS; ++i) y[i].load(p.y, yrow, n0 + lr_piece_col<YT>(i, g), p.N);
  };
  if (n0 < end) fetch();
  if (p.T > 64) lds_barrier();  // the sort's LDS is free

  const int lines = (p.K + 63) / 64, n = lines > wave ? (lines - wave + LR_WAVES - 1) / LR_WAVES : 0;
  const int piece = (lane & 7) ^ (lane >> 3);
  uint32_t off[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = 8 * (i & 1) + (lane >> 3);
    if (i < 2 * XL) {
      const int id = __shfl(rows, r, 64);
      off[i] = (uint32_t)(id >= 0 ? id : row0) * ((uint32_t)p.ldx * E) + (i >> 1) * 128 + 16 * piece;
    } else {
      off[i] = (uint32_t)min(16 * ((i >> 1) - XL) + r, rank - 1) * (uint32_t)p.K * 2 + 16 * piece;
    }
  }
  const char* xb = reinterpret_cast<const char*>(p.x) + wave * 64 * E;
  const char* ab = reinterpret_cast<const char*>(p.a) + ((int64_t)adapter * p.R * p.K + wave * 64) * 2;
  const uint32_t lds0 = lds_addr(&u.ring[wave][0][0]);
  auto issue = [&](int s, int slot) {
    const int k = (s * LR_WAVES + wave) * 64;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint32_t o = off[i];
      if (k + 64 > p.K) {  // a piece past the end of its row: the line's first piece again, masked below
        const int in = (i < 2 * XL ? ((i >> 1) * 128 + 16 * piece) / E : 8 * piece);
        if (k + in >= p.K) o -= (i < 2 * XL ? (i >> 1) * 128 : 0) + 16 * piece;
      }
      dma16(i < 2 * XL ? xb + (int64_t)s * LR_WAVES * 64 * E : ab + (int64_t)s * LR_WAVES * 128, o,
            lds0 + slot * BYTES + i * 1024);
    }
  };
  f32x4 acc[1][RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < n) issue(d, d);
  int slot = 0;
  for (int s = 0; s < n; ++s) {
    const int after = min(D, n - s) - 1;  // stages in flight behind this one
    if (after == 0)
      wait_vmcnt<0>();
    else if (after == 1)
      wait_vmcnt<NI>();
    else if (after == 2)
      wait_vmcnt<2 * NI>();
    else
      wait_vmcnt<3 * NI>();
    asm volatile("" ::: "memory");
    const char* st = u.ring[wave][slot];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Raw<XT> xr[1];
      Raw<WT> ar[RT];
      if constexpr (XT == CCQ_F32) {
        const char* line = st + h * 2048 + c16 * 128;
        xr[0].v[0] = *reinterpret_cast<const u32x4*>(line + (((2 * g) ^ (c16 & 7)) * 16));
        xr[0].v[1] = *reinterpret_cast<const u32x4*>(line + (((2 * g + 1) ^ (c16 & 7)) * 16));
      } else {
        xr[0].v[0] = *reinterpret_cast<const u32x4*>(st + c16 * 128 + (((4 * h + g) ^ (c16 & 7)) * 16));
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
        ar[t].v[0] = *reinterpret_cast<const u32x4*>(st + (XL + t) * 2048 + c16 * 128 + (((4 * h + g) ^ (c16 & 7)) * 16));
      const int left = p.K - ((s * LR_WAVES + wave) * 64 + 32 * h + 8 * g);
      if ((s * LR_WAVES + wave) * 64 + 64 > p.K) {
        lr_fix<XT>(xr[0], 0, 0, left);
#pragma unroll
        for (int t = 0; t < RT; ++t) lr_fix<WT>(ar[t], 0, 0, left);
      }
      lr_multiply<XT, WT, 1, RT>(xr, ar, acc);
    }
    if (s + D < n) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot is read out
      issue(s + D, slot);
    }
    slot = slot == D - 1 ? 0 : slot + 1;
  }
  lds_barrier();
#pragma unroll
  for (int t = 0; t < RT; ++t) u.red[wave][t][lane] = acc[0][t];
  for (int i = threadIdx.x; i < 16 * (32 * RC - 16 * RT); i += LR_THREADS) ps[i & 15][16 * RT + (i >> 4)] = 0.f;
  lds_barrier();
  for (int t = wave; t < RT; t += LR_WAVES) {
    f32x4 s = u.red[0][t][lane];
#pragma unroll
    for (int k = 1; k < LR_WAVES; ++k) s += u.red[k][t][lane];
    // D: column (rank) lane & 15, row (token) 4 (lane >> 4) + i
#pragma unroll
    for (int i = 0; i < 4; ++i) ps[4 * g + i][16 * t + c16] = 16 * t + c16 < rank ? s[i] * scale : 0.f;
  }
  lds_barrier();
  if (n0 >= end) return;
  V pv[RC][PARTS];
  float down = LR_DOWN<WT>;
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
      const float up = lr_pow2(ex);
      down = lr_pow2(-ex);
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
      lr_fix_b<WT>(p, adapter, rank, 32 * c, col, w[c]);
      lr_expand_step<WT, PARTS>(w[c], pv[c], out);
    }
    const float nan = lr_nan_of(out);
    if (__builtin_expect(__any(nan != nan), 0)) {
      // in the wave's part of the ring (p is not scaled here in f16, and the new sums are not finite)
      float(*mine)[64 + 4] = reinterpret_cast<float(*)[64 + 4]>(u.ring[wave][0]);
      lr_lane_exchange();
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(&mine[c16][lr_col<YT>(q, 4 * g)]) = out[q];
      lr_lane_exchange();
      lr_whole_sums<WT, 16>(p, adapter, rank, n0, mine, [&](int i, int r) { return ps[i][r]; });
      lr_lane_exchange();
#pragma unroll
      for (int q = 0; q < 4; ++q) out[q] = *reinterpret_cast<const f32x4*>(&mine[c16][lr_col<YT>(q, 4 * g)]);
    }
    if (own >= 0) lr_store_pieces<YT>(p, y, yrow, n0, g, out, down);
    n0 += 64 * LR_WAVES;
    if (n0 >= end) break;
    fetch();
  }
}

// ------------------------------------------------------------ two kernels --
// A tile's 16 MT tokens, the K range of one split.  RH waves share a K part,
// each with RT * 16 of the ranks (from 16 RT RH blockIdx.z on), so that a
// wave's sums and its loads ahead fit its registers; the K parts' sums meet in
// LDS.
template <int XT, int WT, int MT, int RT, int RH>
__global__ __launch_bounds__(LR_THREADS) void lora_shrink_kernel(const LoraP p) {
  constexpr int TM = 16 * MT, CH = MT == 1 ? 1 : LR_SELF / LR_THREADS;
  constexpr int KP = LR_WAVES / RH;                          // K parts
  constexpr int PASS = MT * RT * RH <= 8 ? MT : 8 / (RT * RH);  // row blocks whose sums are in LDS at once
  __shared__ TileS<TM> tl;
  __shared__ union {
    SortS sort;
    f32x4 red[KP][PASS][RH * RT][64];
  } u;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
  int split;
  const int tile = lr_tile_of(p, split);
  if (tile >= p.tiles) return;
  if (p.meta != nullptr) {
    lr_read_tile<TM>(p, tile, tl);
  } else {
    if (MT == 1 && p.T <= 64) {
      int found;
      const int rows = lr_find_tile_wave(p, tile, found);
      if (threadIdx.x < TM) tl.rows[threadIdx.x] = rows;
      if (threadIdx.x == 0) tl.adapter = found;
      __syncthreads();
    } else {
      lr_find_tile<TM, CH>(p, [&](int) { return tile; }, tl, u.sort);
    }
    if (split == 0 && blockIdx.z == 0 && threadIdx.x < TM)  // for the second kernel
      p.tile_rows[(int64_t)tile * TM + threadIdx.x] = tl.rows[threadIdx.x];
  }
  const int adapter = tl.adapter;
  const int rank = adapter < 0 ? 0 : lr_rank(p, adapter);
  if (split == 0 && blockIdx.z == 0) lr_write_info(p, tile, adapter, rank, p.S);
  const int rz = blockIdx.z * RH * RT * 16;
  if (rz >= rank) return;
  const int h = wave % RH, part = wave / RH, r0 = rz + h * RT * 16;
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
  const int kw = (p.kchunk / 32 + KP - 1) / KP * 32;  // per wave
  const int ks = split * p.kchunk, ke = min(ks + p.kchunk, p.K), k0 = ks + part * kw, k1 = min(k0 + kw, ke);
  if (r0 < rank) {
    if constexpr (MT == 1)
      lr_shrink<XT, WT, MT, RT, (RT == 4 ? 4 : 8) / (XT == CCQ_F32 ? 2 : 1)>(p, xrow, arow, k0, k1, acc);
    else
      lr_shrink_ring<XT, WT, MT, RT, RT == 1 ? 3 : 2>(p, xrow, arow, k0, k1, acc);
  }
#pragma unroll
  for (int m0 = 0; m0 < MT; m0 += PASS) {
    __syncthreads();
#pragma unroll
    for (int m = 0; m < PASS; ++m)
#pragma unroll
      for (int t = 0; t < RT; ++t) u.red[part][m][h * RT + t][lane] = acc[m0 + m][t];
    __syncthreads();
    for (int i = wave; i < PASS * RH * RT; i += LR_WAVES) {
      const int m = i / (RH * RT), t = i - m * (RH * RT);
      if (rz + 16 * t >= rank) continue;  // the workspace's rows end with the last used 16 ranks
      f32x4 s = u.red[0][m][t][lane];
#pragma unroll
      for (int k = 1; k < KP; ++k) s += u.red[k][m][t][lane];
      const int r = rz + 16 * t + c16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // D: column (rank) lane & 15, row (token) 4 (lane >> 4) + e
        const int id = tl.rows[16 * (m0 + m) + 4 * g + e];
        if (id >= 0) p.p[((int64_t)split * p.T + id) * p.Rp + r] = r < rank ? s[e] : 0.f;
      }
    }
  }
}

// The same for 64-token tiles of aligned rows, through LDS: a wave's load then
// takes 8 rows x 128 bytes, whole lines, where the operand loads above ask for
// half lines of 16 rows.  A stage holds 64 Q columns k of the 64 tokens and of
// the RT * 16 ranks, copied by LDS DMA into a ring of D stages, D - 1 ahead;
// each wave multiplies one step of 32 k (part) of it for RTW * 16 ranks (h).
// In a line the 16-byte piece i of row r lies at i ^ (r & 7), so that the
// operand reads of 8 neighbouring lanes cover all banks.
// T=4096 K=14336 R=128: 42.6 us, 2.6 TB/s of x (47 by three splits; then 34
// with x in the last level cache, 27 at R=16).  A, two thirds of a stage, comes
// from L2; more stages ahead, x and A copied by waves of their own, and other
// orders of the stages left the time as it is.
template <int XT, int WT, int RT>
struct TileShrink {
  static constexpr int RTW = RT == 8 ? 4 : RT == 4 ? 2 : 1, RH = RT / RTW, KP = LR_WAVES / RH, Q = KP / 2;
  static constexpr int SK = 64 * Q;                              // k of a stage
  static constexpr int XL = Q * (XT == CCQ_F32 ? 2 : 1);         // lines of a row of x, of A: Q
  static constexpr int X_BYTES = XL * 64 * 128, BYTES = X_BYTES + Q * 16 * RT * 128;
  static constexpr int NI = BYTES / 1024 / LR_WAVES;             // copies of a wave per stage
  static constexpr int FIT = 144 * 1024 / BYTES, D = FIT > 6 ? 6 : FIT;
  static_assert(BYTES % (1024 * LR_WAVES) == 0 && D >= 2 && (D - 2) * NI < 64);
  static_assert(D * BYTES >= KP * 4 * RT * 1024, "the partial sums reuse the ring");
};

template <int XT, int WT, int RT>
__global__ __launch_bounds__(LR_THREADS) void lora_shrink_tile_kernel(const LoraP p) {
  using C = TileShrink<XT, WT, RT>;
  constexpr int RTW = C::RTW, RH = C::RH, KP = C::KP, NI = C::NI, D = C::D;
  constexpr int E = XT == CCQ_F32 ? 4 : 2;
  __shared__ TileS<64> tl;
  __shared__ __align__(16) union {
    SortS sort;
    char ring[D][C::BYTES];
    f32x4 red[KP][4][RT][64];
  } u;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
  // the tiles' K ranges, range by range, in eight parts of one size, one to an
  // XCD: its L2 then reads few adapters' A, and of those one range each
  int split = 0, tile = -1, total = 0, S = p.S, kchunk = p.kchunk;
  auto pick = [&](int count) {
    total = count;
    if (count <= p.few) {
      S = p.S_few;
      kchunk = p.kchunk_few;
    }
    const int xcd = blockIdx.x & 7, all = count * S, from = (int)((int64_t)xcd * all >> 3);
    const int at = from + (blockIdx.x >> 3);
    if (at < (int)((int64_t)(xcd + 1) * all >> 3)) {
      split = at / count;
      tile = at - split * count;
    }
    return tile;
  };
  if (p.meta != nullptr) {
    pick(p.meta[0]);
    if (tile >= 0) lr_read_tile<64>(p, tile, tl);
  } else {
    lr_find_tile<64, LR_SELF / LR_THREADS>(p, pick, tl, u.sort);
    if (tile >= 0 && split == 0 && blockIdx.z == 0 && threadIdx.x < 64)  // for the second kernel
      p.tile_rows[(int64_t)tile * 64 + threadIdx.x] = tl.rows[threadIdx.x];
  }
  if (blockIdx.x == 0 && blockIdx.z == 0)  // no such tiles
    for (int i = total + threadIdx.x; i < p.tiles; i += LR_THREADS) p.tile_info[i] = make_int4(-1, 0, 0, 0);
  if (tile < 0) return;
  const int adapter = __builtin_amdgcn_readfirstlane(tl.adapter);
  const int rank = __builtin_amdgcn_readfirstlane(adapter < 0 ? 0 : lr_rank(p, adapter));
  if (split == 0 && blockIdx.z == 0) lr_write_info(p, tile, adapter, rank, S);
  const int rz = blockIdx.z * RT * 16;
  if (rz >= rank) return;
  const int ks = split * kchunk, ke = min(ks + kchunk, p.K), stages = (ke - ks + C::SK - 1) / C::SK;

  // copy i of the wave: 8 rows of one line, this lane piece `piece` of row `row`
  uint32_t off[NI];   // bytes from the base below, at the split's first stage
  const int piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = wave * NI + i;
    if (c < C::X_BYTES / 1024) {
      const int own = tl.rows[(c & 7) * 8 + (lane >> 3)];
      off[i] = (uint32_t)(own >= 0 ? own : tl.rows[0]) * ((uint32_t)p.ldx * E) + (c >> 3) * 128 + 16 * piece;
    } else {
      const int a = c - C::X_BYTES / 1024, r = rz + (a % (2 * RT)) * 8 + (lane >> 3);
      off[i] = (uint32_t)min(r, rank - 1) * (uint32_t)p.K * 2 + a / (2 * RT) * 128 + 16 * piece;
    }
  }
  const char* xb = reinterpret_cast<const char*>(p.x) + (int64_t)ks * E;
  const char* ab = reinterpret_cast<const char*>(p.a) + ((int64_t)adapter * p.R * p.K + ks) * 2;
  const uint32_t lds0 = lds_addr(&u);
  auto issue = [&](int s, int slot) {
    const bool tail = ks + (s + 1) * C::SK > p.K;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = wave * NI + i;
      const bool is_x = c < C::X_BYTES / 1024;
      uint32_t o = off[i];
      if (tail) {  // a piece past the end of its row: the row's first piece of the stage again, masked below
        const int e = is_x ? E : 2, line = is_x ? c >> 3 : (c - C::X_BYTES / 1024) / (2 * RT);
        if (ks + s * C::SK + (line * 128 + 16 * piece) / e >= p.K) o -= line * 128 + 16 * piece;
      }
      dma16((is_x ? xb + (int64_t)s * C::SK * E : ab + (int64_t)s * C::SK * 2), o, lds0 + slot * C::BYTES + c * 1024);
    }
  };
  const int h = wave % RH, part = wave / RH;
  f32x4 acc[4][RTW];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int t = 0; t < RTW; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();  // the sort's LDS is free
#pragma unroll
  for (int d = 0; d < D - 1; ++d) issue(min(d, stages - 1), d);
  int slot = 0;
  for (int s = 0; s < stages; ++s) {
    wait_vmcnt<(D - 2) * NI>();
    lds_barrier();  // stage s is in LDS for all, and the slot before it is read out
    issue(min(s + D - 1, stages - 1), slot == 0 ? D - 1 : slot - 1);  // past the range: not read
    const char* st = u.ring[slot];
    Raw<XT> xr[4];
    Raw<WT> ar[RTW];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int row = 16 * m + c16;
      if constexpr (XT == CCQ_F32) {
        const char* line = st + part * 8192 + row * 128;
        xr[m].v[0] = *reinterpret_cast<const u32x4*>(line + (((2 * g) ^ (row & 7)) * 16));
        xr[m].v[1] = *reinterpret_cast<const u32x4*>(line + (((2 * g + 1) ^ (row & 7)) * 16));
      } else {
        xr[m].v[0] = *reinterpret_cast<const u32x4*>(st + (part >> 1) * 8192 + row * 128 +
                                                     (((4 * (part & 1) + g) ^ (row & 7)) * 16));
      }
    }
#pragma unroll
    for (int t = 0; t < RTW; ++t) {
      const int row = 16 * (h * RTW + t) + c16;
      ar[t].v[0] = *reinterpret_cast<const u32x4*>(st + C::X_BYTES + (part >> 1) * (16 * RT * 128) + row * 128 +
                                                   (((4 * (part & 1) + g) ^ (row & 7)) * 16));
    }
    const int left = p.K - (ks + s * C::SK + 32 * part + 8 * g);
    if (ks + (s + 1) * C::SK > p.K) {
#pragma unroll
      for (int m = 0; m < 4; ++m) lr_fix<XT>(xr[m], 0, 0, left);
#pragma unroll
      for (int t = 0; t < RTW; ++t) lr_fix<WT>(ar[t], 0, 0, left);
    }
    lr_multiply<XT, WT, 4, RTW>(xr, ar, acc);
    slot = slot == D - 1 ? 0 : slot + 1;
  }
  wait_vmcnt<0>();
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int t = 0; t < RTW; ++t) u.red[part][m][h * RTW + t][lane] = acc[m][t];
  __syncthreads();
  for (int i = wave; i < 4 * RT; i += LR_WAVES) {
    const int m = i / RT, t = i % RT;
    if (rz + 16 * t >= rank) continue;  // the workspace's rows end with the last used 16 ranks
    f32x4 s = u.red[0][m][t][lane];
#pragma unroll
    for (int k = 1; k < KP; ++k) s += u.red[k][m][t][lane];
    const int r = rz + 16 * t + c16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // D: column (rank) lane & 15, row (token) 4 (lane >> 4) + e
      const int id = tl.rows[16 * m + 4 * g + e];
      if (id >= 0) p.p[((int64_t)split * p.T + id) * p.Rp + r] = r < rank ? s[e] : 0.f;
    }
  }
}

// A tile's 16 MT tokens, ncols columns: p summed over the splits, scaled and
// in parts in LDS; a wave then takes 64 columns of 16 MP tokens at a time.  The
// products' lanes hold 4 columns of 16 tokens each: they pass through the
// wave's part of LDS into rows, so that y is read and written in whole lines
// (8 lanes a row of 128 bytes).  A block's weights, up to KEEP chunks of 32
// ranks, stay in registers for all tokens of the tile, each chunk replaced by
// the next block's behind its last product (more than 128 ranks pass through
// as a stream); y of the next step is loaded before the products of this one.
// p's loads go first: a wave waits for its loads in order, and those of y come
// from HBM.  T=2048 N=14336 R=16: 25.7 us for 117 MB of y (4.6 TB/s; 27.5 with
// y before p, 30.1 with the weights loaded step by step).  T=4096 N=4096
// R=128: 30.8 us, 10 of them until p of its splits is in LDS.
template <int WT, int YT, int MT, int KEEP>
__global__ __launch_bounds__(LE_THREADS, YT == CCQ_F32 || KEEP * MT >= (MT == 1 ? 4 : 8) ? 2 : 3) void lora_expand_kernel(
    const LoraP p) {
  using V = typename Half<WT>::vec;
  constexpr int PARTS = WT == CCQ_F16 ? 2 : YT == CCQ_F32 ? 3 : 2, TM = 16 * MT, WAVES = LE_THREADS / 64;
  constexpr int MP = MT < 2 ? MT : 2, PAIRS = MT / MP;
  constexpr bool STREAM = KEEP > 4;
  constexpr int SLOTS = !STREAM ? KEEP : YT == CCQ_F32 ? 2 : 4;
  constexpr int E = YT == CCQ_F32 ? 4 : 2, COLS = 16 / E, RL = 64 / COLS;  // lanes of a row
  constexpr int RI = 64 / RL, YN = 16 * MP / RI;                           // rows of an access, accesses of a step
  __shared__ TileS<TM> tl;
  __shared__ float downs[TM];
  // (with half of it two workgroups of three parts and 128 ranks fit a CU: T=3020 N=5152 float32 68 -> 50 us)
  constexpr int TURN = YT == CCQ_F32 && KEEP == 4 && MT > 1 ? 1 : MP;  // row blocks that turn at once
  __shared__ __align__(16) float turn[WAVES][16 * TURN][64 + 4];
  extern __shared__ __align__(16) uint16_t parts[];  // [PARTS][TM][ld]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
  const int yr = lane / RL, yc = lane % RL * COLS;  // this lane's row and columns of an access to y
  const int tile = blockIdx.x % p.tiles, group = blockIdx.x / p.tiles;
  const int4 info = p.tile_info[tile];
  if (threadIdx.x < TM) tl.rows[threadIdx.x] = p.tile_rows[(int64_t)tile * TM + threadIdx.x];
  __syncthreads();
  const int adapter = info.x, rank = info.y;
  if (adapter < 0) return;
  const float scale = __int_as_float(info.z) / LR_DOWN<WT>;
  const int rc = (rank + 31) / 32, r16 = (rank + 15) & ~15, ld = 32 * rc + 8;
  const int first = group * p.ncols + 64 * wave, end = min((group + 1) * p.ncols, p.N);
  const int blocks = first < end ? (end - first + 64 * WAVES - 1) / (64 * WAVES) : 0, steps = blocks * PAIRS;
  YPiece<YT> y[2][YN];
  Raw<WT> w[SLOTS][4];  // the block's weights in chunks of 32 ranks
  auto block_of = [&](int step) { return first + 64 * WAVES * (step / PAIRS); };  // step = block * PAIRS + pair
  auto load_b = [&](int n0, int c, Raw<WT>(&v)[4]) {
    lr_load_b<WT>(p, adapter, 32 * c, [&](int q) { return n0 + 16 * q + c16; }, v);
  };
  auto fetch = [&](int step, YPiece<YT>(&v)[YN]) {
    const int m0 = (step % PAIRS) * MP;
#pragma unroll
    for (int i = 0; i < YN; ++i) {
      const int id = tl.rows[16 * m0 + RI * i + yr];
      v[i].load(p.y, (int64_t)(id >= 0 ? id : tl.rows[0]) * p.ldy, block_of(step) + yc, p.N);
    }
  };
  // 4 ranks a lane, as many lanes a row as its ranks take.  A tile of 16 rows may leave waves: they share the splits,
  // the first ones adding the shares in order.
  const int lp = r16 <= 16 ? 2 : r16 <= 32 ? 3 : r16 <= 64 ? 4 : r16 <= 128 ? 5 : 6;
  const int j = threadIdx.x & ((1 << lp) - 1), sub = threadIdx.x >> lp;
  const bool spare = MT == 1 && lp < 4;
  const int share = spare ? __builtin_amdgcn_readfirstlane(sub >> 4) : 0, shares = spare ? 16 >> lp : 1;
  const int S = __builtin_amdgcn_readfirstlane(info.w);
  const int per = S <= 4 ? S : (S + shares - 1) / shares, s0 = share * per, s1 = min(s0 + per, S);
  const int rows = spare ? 16 : LE_THREADS >> lp, passes = TM / rows, row0 = spare ? sub & 15 : sub;
  float* shared = reinterpret_cast<float*>(parts + PARTS * TM * ld);  // [shares][16][r16]
  const char* pb = reinterpret_cast<const char*>(p.p);
  const int64_t pstep = (int64_t)p.T * p.Rp * 4;
  constexpr int HELD = MT > 1 && (KEEP == 1 || KEEP == 4 && YT == CCQ_F32) ? 8 : 16;  // (more would spill)
  constexpr int U = MT == 1 ? 1 : KEEP == 1 || HELD == 8 ? 2 : 4, KS = HELD / U;  // passes and splits whose loads are in flight together
  f32x4 o[U][KS];
  auto load_p = [&](int pass, int s) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (pass + u < passes) {
        const int id = tl.rows[(pass + u) * rows + row0];
        const uint32_t off = ((uint32_t)(id >= 0 ? id : tl.rows[0]) * (uint32_t)p.Rp + (4 * j < r16 ? 4 * j : 0)) * 4;
#pragma unroll
        for (int k = 0; k < KS; ++k)
          if (s + k < s1) o[u][k] = *reinterpret_cast<const f32x4*>(pb + (s + k) * pstep + off);
      }
  };
  load_p(0, s0);
  if (steps > 0) {
    fetch(0, y[0]);
#pragma unroll
    for (int c = 0; c < SLOTS; ++c)
      if (c < rc) load_b(first, c, w[c]);
  }
#pragma unroll 1
  for (int pass = 0; pass < passes; pass += U) {
    f32x4 sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s = s0; s < s1; s += KS) {
      if (s > s0) load_p(pass, s);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        if (s + k < s1) {
#pragma unroll
          for (int u = 0; u < U; ++u) sum[u] += o[u][k];
        }
    }
    if (pass + U < passes) load_p(pass + U, s0);
    if constexpr (MT == 1) {
      if (spare && S > 4) {  // else the first share is all
        if (share > 0 && 4 * j < r16) *reinterpret_cast<f32x4*>(shared + (share * 16 + row0) * r16 + 4 * j) = sum[0];
        lds_barrier();
        if (share == 0 && 4 * j < r16)
          for (int k = 1; k < shares; ++k) sum[0] += *reinterpret_cast<const f32x4*>(shared + (k * 16 + row0) * r16 + 4 * j);
      }
      if (share > 0) break;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (pass + u >= passes) break;
      const int row = (pass + u) * rows + row0, id = tl.rows[row];
      float v[4], m = 0.f, up = 1.f, down = LR_DOWN<WT>;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = id >= 0 && 4 * j + e < rank ? sum[u][e] * scale : 0.f;
        m = isfinite(v[e]) ? fmaxf(m, fabsf(v[e])) : m;
      }
      if constexpr (WT == CCQ_F16) {
        for (int off = 1; off < 1 << lp; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const int ex = lr_exponent(m);
        up = lr_pow2(ex);
        down = lr_pow2(-ex);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= up;
      }
      if (j == 0) downs[row] = down;
      if (4 * j < 32 * rc) {
        typename Half<WT>::quad pv[PARTS];
        lr_split<WT, PARTS>(v, pv);
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
          uint16_t* to = parts + (k * TM + row) * ld + 4 * j;
          *reinterpret_cast<typename Half<WT>::quad*>(to) = pv[k];
          if (r16 == 16) *reinterpret_cast<uint64_t*>(to + 16) = 0;  // the chunk's other half
        }
      }
    }
  }
  lds_barrier();
  float(*mine)[64 + 4] = turn[wave];
  for (int s = 0; s < steps; s += 2) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int step = s + d;
      if (step >= steps) break;
      const int next = step + 1 < steps ? step + 1 : step;  // (the last one's again: not used)
      fetch(next, y[d ^ 1]);
      __builtin_amdgcn_sched_barrier(0);
      const int n0 = block_of(step), m0 = (step % PAIRS) * MP;
      f32x4 acc[MP][4];
#pragma unroll
      for (int m = 0; m < MP; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][q] = f32x4{0.f, 0.f, 0.f, 0.f};
      const bool fresh = PAIRS == 1 || d == 0, last = PAIRS == 1 || d == 1;  // of the block's pairs
#pragma unroll 1
      for (int c0 = 0; c0 < (STREAM ? rc : 1); c0 += SLOTS) {
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
          const int c = c0 + j;
          if (c < rc) {
            if (STREAM || fresh) lr_fix_b<WT>(p, adapter, rank, 32 * c, [&](int q) { return n0 + 16 * q + c16; }, w[j]);
#pragma unroll
            for (int m = 0; m < MP; ++m) {
              V pv[PARTS];
#pragma unroll
              for (int k = 0; k < PARTS; ++k)
                pv[k] = *reinterpret_cast<const V*>(parts + (k * TM + 16 * (m0 + m) + c16) * ld + 32 * c + 8 * g);
              lr_expand_step<WT, PARTS>(w[j], pv, acc[m]);
            }
          }
          if (STREAM && c + SLOTS < rc)
            load_b(n0, c + SLOTS, w[j]);
          else if ((STREAM || last) && c0 + SLOTS >= rc && j < rc && step + 1 < steps)
            load_b(block_of(step + 1), j, w[j]);
        }
      }
#pragma unroll
      for (int h = 0; h < MP; h += TURN) {
        lr_lane_exchange();
#pragma unroll
        for (int m = 0; m < TURN; ++m)
#pragma unroll
          for (int q = 0; q < 4; ++q) *reinterpret_cast<f32x4*>(&mine[16 * m + c16][16 * q + 4 * g]) = acc[h + m][q];
        float nan = 0.f;
#pragma unroll
        for (int m = 0; m < TURN; ++m) nan += lr_nan_of(acc[h + m]);
        lr_lane_exchange();
        if (__builtin_expect(__any(nan != nan), 0)) {
          const uint16_t* of = parts + 16 * (m0 + h) * ld;
          lr_whole_sums<WT, 16 * TURN>(p, adapter, rank, n0, mine,
                                       [&](int i, int r) { return lr_join<WT, PARTS>(of + i * ld + r, TM * ld); });
          lr_lane_exchange();
        }
#pragma unroll
        for (int i = 0; i < YN * TURN / MP; ++i) {
          const int at = h * YN / MP + i, row = RI * i + yr, id = tl.rows[16 * (m0 + h) + row];
          float add[COLS];
          const float f = downs[16 * (m0 + h) + row];
#pragma unroll
          for (int e = 0; e < COLS; e += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(&mine[row][yc + e]);
#pragma unroll
            for (int k = 0; k < 4; ++k) add[e + k] = v[k] * f;
          }
          if (id >= 0) y[d][at].add_store(p.y, p.y_dtype, (int64_t)id * p.ldy, n0 + yc, p.N, add);
        }
      }
    }
  }
}

// Buffers of fewer than 8 values (no 16-byte load fits them), so K, N or both
// are below 8: a workgroup forms a token's p, a wave for each rank, then takes
// its 256 columns.  Sums in 64 bits.
__device__ __forceinline__ float lr_value(const void* v, int64_t i, int dt) {
  if (dt == CCQ_F32) return reinterpret_cast<const float*>(v)[i];
  const uint32_t u = reinterpret_cast<const uint16_t*>(v)[i];
  return dt == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
}
__global__ __launch_bounds__(256) void lora_tiny_kernel(const LoraP p, int x_dtype, int w_dtype) {
  __shared__ double ps[LR_MAX_R];
  const int64_t token = blockIdx.x, n = (int64_t)blockIdx.y * 256 + threadIdx.x;
  const int64_t adapter = p.index[token];
  if (adapter < 0 || adapter >= p.L) return;
  const int rank = lr_rank(p, (int)adapter), lane = threadIdx.x & 63;
  if (rank == 0) return;
  for (int r = threadIdx.x >> 6; r < rank; r += 4) {
    double sum = 0;
    for (int k = lane; k < p.K; k += 64)
      sum += (double)lr_value(p.x, token * p.ldx + k, x_dtype) *
             (double)lr_value(p.a, (adapter * p.R + r) * p.K + k, w_dtype);
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (lane == 0) ps[r] = sum;
  }
  __syncthreads();
  if (n >= p.N) return;
  double sum = 0;
  for (int r = 0; r < rank; ++r) sum += ps[r] * (double)lr_value(p.b, (adapter * p.N + n) * p.R + r, w_dtype);
  const int64_t at = token * p.ldy + n;
  const float v = (float)(lr_value(p.y, at, p.y_dtype) + sum * (p.scale != nullptr ? p.scale[adapter] : 1.f));
  if (p.y_dtype == CCQ_F32)
    reinterpret_cast<float*>(p.y)[at] = v;
  else
    reinterpret_cast<uint16_t*>(p.y)[at] =
        (uint16_t)(p.y_dtype == CCQ_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
}

size_t a256l(size_t b) { return (b + 255) & ~(size_t)255; }

struct LoraPlan {
  bool fused, align;
  int64_t tm, tiles, S, kchunk, Rp, ncols;
  int64_t few, S_few, kchunk_few;  // as in LoraP
  size_t off_rows, off_tile, off_info, off_meta, off_counts, off_align, off_p, total;
};

// Of a tile's x and A, which each workgroup of the one kernel reads.  One
// kernel and two, in us: T=16 K=4096 N=14336 R=16 (256 KiB) 8.6 and 11.8, T=64
// K=N=4096 R=32 (384) 8.3 and 10.4, T=1 K=N=8192 R=16 (512) 10.2 and 9.3, T=16
// K=14336 N=4096 R=16 (896) 14.3 and 10.8.
constexpr int64_t LR_FUSED_BYTES = 384 << 10;

// lines: lora_lines, one_type: x float32 or of A's type
LoraPlan lora_plan(int64_t T, const ccq_lora_adapters* ad, bool lines, bool one_type, bool x32) {
  LoraPlan L = {};
  const int64_t K = ad->in_features, N = ad->out_features, R = ad->rank_max;
  L.Rp = cdiv(R, 16) * 16;
  L.fused = lines && one_type && T <= LR_THREADS && R <= 32 && (16 + L.Rp) * K * 2 <= LR_FUSED_BYTES;
  L.align = T > LR_SELF;
  // tiles of 16 up to a token a thread of the sort (T=256 K=N=4096 R=64 14.3 us, by tiles of 64 19.0; T=512 18.6 and
  // 20.0), of 64 above, which read A a quarter as often
  L.tm = T <= LR_THREADS ? 16 : 64;
  L.tiles = ccq_moe_align_max_tiles(T, ad->num_adapters, L.tm);
  if (L.tiles > T) L.tiles = T;  // every tile has a token
  // columns per workgroup: 64 for each wave, or a multiple where that still fills the CUs
  const int64_t unit = L.fused ? 64 * LR_WAVES : LE_THREADS;
  const int64_t likely = L.tm == 16 ? L.tiles : cdiv(T, L.tm) + (L.tiles - cdiv(T, L.tm)) / 2;
  // (a workgroup of one kernel fills a CU; three, two or one of the expand kernel fit, by registers and LDS.  A second
  // round for a part of them is what costs: T=2048 N=14336 R=64 35 us by groups for two a CU, 46 for three; T=4096
  // N=4096 R=256 59 for one, 70 for two; T=4096 N=4096 R=128 34 by 8 groups of 512 columns, 43 by 6 of 768)
  const int64_t slots = L.fused ? 256 : L.tm == 16 ? (R <= 64 ? 768 : 512) : R <= 32 ? 768 : R <= 128 ? 512 : 256;
  const int64_t want = L.fused ? slots / likely : (slots + likely / 2) / likely;
  int64_t groups = cdiv(N, unit);
  if (groups > want) groups = want < 1 ? 1 : want;
  L.ncols = cdiv(cdiv(N, groups), unit) * unit;
  if (L.fused) {
    L.S = 1;
    return L;
  }
  // splits of K: for 16-token tiles (whose A is read once) as many as give every CU a workgroup, and no more than where
  // p's reading grows faster than K's parts shrink (S^2 R = 3.5 K: T=100 K=4560 N=400 R=128 10 splits 18.1 us, 18 20.6; T=30
  // K=N=8192 R=256 10 27.4, 32 33.8); else (one workgroup fits a CU) the fewest within 5% of the shortest time, in units of
  // a k: the rounds of the CUs, each as long as its part of K and a start worth 512, and each split's p, which every
  // group of columns reads (T=1000 K=N=4096 R=128 32.2 us, without this term 33.8; R=200 46 and 50).  float32 x takes
  // four times as long a k (its products are the 32-bit ones; T=1051 K=2352 R=128 48 us, at 16-bit costs 61).
  int64_t S = 1;
  if (L.tm == 16) {
    S = 256 / likely < cdiv(K, 256) ? 256 / likely : cdiv(K, 256);
    S = S > 32 ? 32 : S;
    while (S > 1 && 2 * S * S * L.Rp > 7 * K) --S;
    S = S < 1 ? 1 : S;
  } else {
    const int64_t most = cdiv(K, LR_WAVES * 64) < 8 ? cdiv(K, LR_WAVES * 64) : 8;
    const int64_t part = (R < 64 ? R : R < 128 ? 64 : 128) / (x32 ? 4 : 1), start = x32 ? 128 : 512;
    auto splits = [&](int64_t tiles) {
      auto time = [&](int64_t s) { return (double)cdiv(tiles * s, 256) * ((double)K / s + start) + (double)(s * part); };
      double best = time(1);
      for (int64_t s = 2; s <= most; ++s) best = time(s) < best ? time(s) : best;
      int64_t s = 1;
      while (time(s) > 1.05 * best) ++s;
      return s;
    };
    S = splits(likely);
    // where few tiles are padding the kernel, which counts them, may take more in as many rounds (T=4096 K=14336 R=128,
    // 62 tiles of at most 68: 4 splits 42.6 us, 3 46.9)
    const int64_t least = cdiv(T, L.tm), S_few = lines ? splits(least) : S;
    if (S_few > S) {
      L.kchunk_few = cdiv(cdiv(K, S_few), 256) * 256;
      L.S_few = cdiv(K, L.kchunk_few);
      L.few = cdiv(least * L.S_few, 256) * 256 / L.S_few;
    }
  }
  const int64_t step = L.tm == 16 ? 32 : 256;  // the largest stage of a 64-token tile
  L.kchunk = cdiv(cdiv(K, S), step) * step;
  L.S = cdiv(K, L.kchunk);
  size_t o = 0;
  L.off_rows = o;
  o += a256l((size_t)L.tiles * L.tm * 4);
  L.off_info = o;
  o += a256l((size_t)L.tiles * sizeof(int4));
  L.off_tile = o;
  if (L.align) o += a256l((size_t)L.tiles * 4);
  L.off_meta = o;
  o += 256;
  L.off_counts = o;
  if (L.align) o += a256l((size_t)ad->num_adapters * 4);
  L.off_align = o;
  if (L.align) o += a256l(align_scratch_bytes(T, ad->num_adapters));
  L.off_p = o;
  o += a256l((size_t)std::max(L.S, L.S_few) * T * L.Rp * 4);
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
  const dim3 grid((unsigned)(((p.tiles + 7) & ~7) * groups)), block(LR_THREADS);
  if (p.R <= 16)
    launch((lora_fused_kernel<XT, WT, YT, 1>), grid, block, 0, st, p);
  else
    launch((lora_fused_kernel<XT, WT, YT, 2>), grid, block, 0, st, p);
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
  const dim3 grid((unsigned)(((p.tiles + 7) & ~7) * p.S), 1, (unsigned)cdiv(rt, 8)), block(LR_THREADS);
  if (rt <= 1)
    launch((lora_shrink_kernel<XT, WT, MT, 1, 1>), grid, block, 0, st, p);
  else if (rt <= 2)
    launch((lora_shrink_kernel<XT, WT, MT, 2, 1>), grid, block, 0, st, p);
  else if (rt <= 4)
    launch((lora_shrink_kernel<XT, WT, MT, 4, 1>), grid, block, 0, st, p);
  else
    launch((lora_shrink_kernel<XT, WT, MT, 4, 2>), grid, block, 0, st, p);
}

// 64-token tiles whose rows' 16-byte pieces are aligned
template <int XT, int WT>
void shrink_tile_launch(const LoraP& p, hipStream_t st) {
  const int rt = (int)cdiv(p.R, 16);
  const dim3 grid((unsigned)(((p.tiles + 7) & ~7) * std::max(p.S, p.S_few)), 1, (unsigned)cdiv(rt, 8)), block(LR_THREADS);
  if (rt <= 1)
    launch((lora_shrink_tile_kernel<XT, WT, 1>), grid, block, 0, st, p);
  else if (rt <= 2)
    launch((lora_shrink_tile_kernel<XT, WT, 2>), grid, block, 0, st, p);
  else if (rt <= 4)
    launch((lora_shrink_tile_kernel<XT, WT, 4>), grid, block, 0, st, p);
  else
    launch((lora_shrink_tile_kernel<XT, WT, 8>), grid, block, 0, st, p);
}
template <int WT, int MT, int KEEP>
void expand_launch(const LoraP& p, int64_t groups, hipStream_t st) {
  const dim3 grid((unsigned)(p.tiles * groups)), block(LE_THREADS);
  const size_t ld = (size_t)cdiv(p.R, 32) * 32 + 8, part = ld * 16 * MT * 2;
  const size_t shared = MT == 1 && p.S > 4 ? 4 * 16 * 16 * 4 : 0;  // 4 shares of up to 16 ranks, 2 of up to 32
  if (p.y_dtype == CCQ_F32)
    launch((lora_expand_kernel<WT, CCQ_F32, MT, KEEP>), grid, block, part * (WT == CCQ_BF16 ? 3 : 2) + shared, st, p);
  else
    launch((lora_expand_kernel<WT, CCQ_BF16, MT, KEEP>), grid, block, part * 2 + shared, st, p);
}

template <int WT, int MT>
int two_launches(const LoraP& p, int x_dtype, bool lines, int64_t groups, hipStream_t st) {
  if (MT == 4 && lines) {
    if (x_dtype == CCQ_BF16)
      shrink_tile_launch<CCQ_BF16, WT>(p, st);
    else if (x_dtype == CCQ_F16)
      shrink_tile_launch<CCQ_F16, WT>(p, st);
    else
      shrink_tile_launch<CCQ_F32, WT>(p, st);
  } else if (x_dtype == CCQ_BF16)
    shrink_launch<CCQ_BF16, WT, MT>(p, st);
  else if (x_dtype == CCQ_F16)
    shrink_launch<CCQ_F16, WT, MT>(p, st);
  else
    shrink_launch<CCQ_F32, WT, MT>(p, st);
  if (int rc = launch_status("ccq_lora_add (shrink)")) return rc;
  if (p.R <= 32)
    expand_launch<WT, MT, 1>(p, groups, st);
  else if (p.R <= 64)
    expand_launch<WT, MT, 2>(p, groups, st);
  else if (p.R <= 128)
    expand_launch<WT, MT, 4>(p, groups, st);
  else
    expand_launch<WT, MT, 8>(p, groups, st);
  return launch_status("ccq_lora_add (expand)");
}

bool lora_float_code(int dt) { return dt == CCQ_F32 || dt == CCQ_F16 || dt == CCQ_BF16; }
// rows of x and A aligned to 16 bytes, x within 32-bit offsets
bool lora_lines(const void* x, int x_dtype, int64_t ldx, int64_t T, const ccq_lora_adapters* ad) {
  const int64_t e = x_dtype == CCQ_F32 ? 4 : 2;
  return ad->in_features % 8 == 0 && aligned(x, 16) && aligned(ad->a, 16) && ldx * e % 16 == 0 &&
         ldx <= ((int64_t)1 << 32) / (T * e) - 1;
}
bool lora_one_type(int x_dtype, const ccq_lora_adapters* ad) { return x_dtype == CCQ_F32 || x_dtype == ad->dtype; }

}  // namespace

}  // namespace ccq

using namespace ccq;

extern "C" size_t ccq_lora_workspace_size(const void* x, int x_dtype, int64_t ldx, int64_t T,
                                          const ccq_lora_adapters* ad) {
  if (T <= 0 || T > 65536 || !lora_float_code(x_dtype) || check_adapters(ad, "ccq_lora_workspace_size")) return 0;
  return lora_plan(T, ad, lora_lines(x, x_dtype, ldx, T, ad), lora_one_type(x_dtype, ad), x_dtype == CCQ_F32).total;
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
  const bool lines = lora_lines(x, x_dtype, ldx, T, ad);
  const LoraPlan L = lora_plan(T, ad, lines, lora_one_type(x_dtype, ad), x_dtype == CCQ_F32);
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
  p.few = (int)L.few;
  p.S_few = (int)L.S_few;
  p.kchunk_few = (int)L.kchunk_few;
  p.tiles = (int)L.tiles;
  p.ncols = (int)L.ncols;
  p.y_dtype = y_dtype;
  p.last_x = (T - 1) * ldx + p.K - 8;
  p.last_a = ad->num_adapters * ad->rank_max * ad->in_features - 8;
  p.last_b = ad->num_adapters * ad->rank_max * ad->out_features - 8;
  if (p.last_x < 0 || p.last_a < 0 || p.last_b < 0) {
    launch(lora_tiny_kernel, dim3((unsigned)T, (unsigned)cdiv(p.N, 256)), dim3(256), 0, st, p, x_dtype, ad->dtype);
    return launch_status("ccq_lora_add");
  }
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
  p.tile_info = (int4*)(ws + L.off_info);
  p.p = (float*)(ws + L.off_p);
  if (L.align) {
    p.meta = (const int32_t*)(ws + L.off_meta);
    const int rc = launch_align(index, T, p.L, L.tm, p.tile_rows, p.tile_adapter, (int32_t*)(ws + L.off_meta),
                                (int32_t*)(ws + L.off_counts), st, ws + L.off_align, align_scratch_bytes(T, p.L));
    if (rc) return rc;
  }
  if (ad->dtype == CCQ_BF16)
    return L.tm == 16 ? two_launches<CCQ_BF16, 1>(p, x_dtype, lines, groups, st)
                      : two_launches<CCQ_BF16, 4>(p, x_dtype, lines, groups, st);
  return L.tm == 16 ? two_launches<CCQ_F16, 1>(p, x_dtype, lines, groups, st)
                    : two_launches<CCQ_F16, 4>(p, x_dtype, lines, groups, st);
}
