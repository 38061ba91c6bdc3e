// Linears with weights of 16 bits and an epilogue, for a batch of rows and for
// rows grouped by expert:
//   z = x w^T + bias,   y = act(z) + residual,
//   gated (w holds 2N rows):   y = act(z[:, :N]) * z[:, N:] + residual,
// x [M, K], w [N, K] (grouped: w[e] for the rows offsets[e] .. offsets[e + 1] - 1),
// products and everything after them in float32, y rounded once.
//
// Both kernels give the matrix instructions w as their first operand, so a lane
// ends with four neighbouring columns of one row of y, and with the gate and up
// rows of w in turn (16 by 16) also both halves of a gated value: the epilogue
// needs no exchange.
//
// dense_few_kernel   up to 64 rows at once: w goes from memory to registers, the
//                    waves of a workgroup share K and add up at the end.
// dense_tile_kernel  tiles of rows and columns through LDS.
#include "ccq_common.h"

#include <algorithm>
#include <type_traits>

namespace ccq {

namespace {

constexpr int64_t DN_MAX_E = 1024;

struct DenseP {
  const void* x;
  const void* w;
  const void* bias;       // or null
  const void* residual;   // or null
  void* y;
  float* part;            // [splits][M][W] sums of K's splits, or null
  const int32_t* offsets; // grouped, or null
  int64_t ldx, ldr, ldy;
  int64_t M;              // rows in all
  int K, N, W;            // W: rows of w, N or 2N
  int E;
  int gated, act, bias_dtype, y_dtype;
  int mtiles, ntiles;     // most row tiles, column tiles
  int splits, kchunk;     // K's splits, K of each (whole stages)
};

template <int DT>
struct DnVec {
  using type = bf16x8;
};
template <>
struct DnVec<CCQ_F16> {
  using type = f16x8;
};

__device__ __forceinline__ f32x4 dn_mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 dn_mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ------------------------------------------------------------- epilogue --
__device__ __forceinline__ float dn_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ float dn_rcp(float v) { return __builtin_amdgcn_rcpf(v); }

// z Phi(z): Phi(-|z|) = exp(-x^2) erfcx(x) / 2 with x = |z| / sqrt 2 and erfcx
// a polynomial in t = 1 / (1 + 0.33 x) without a constant term, fitted over
// x <= 10 to 9.4e-8 of its value (beyond, exp(-x^2) is 0 in float32).  Both tails
// keep their relative accuracy, and it takes a third of erff's instructions.
__device__ __forceinline__ float dn_gelu(float z) {
  const float x = fabsf(z) * 0.707106781f;
  const float t = dn_rcp(fmaf(0.33f, x, 1.f));
  float q = fmaf(t, -0.1353449f, 0.46023397f);
  q = fmaf(t, q, -0.35114448f);
  q = fmaf(t, q, 0.40849535f);
  q = fmaf(t, q, 0.04722303f);
  q = fmaf(t, q, 0.20122319f);
  q = fmaf(t, q, 0.18295605f);
  q = fmaf(t, q, 0.1863578f);
  q = q * t * 0.5f * dn_exp(-x * x);
  return z * (z >= 0.f ? 1.f - q : q);
}

__device__ __forceinline__ float dn_act(int act, float z) {
  if (act == CCQ_ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == CCQ_ACT_GELU) return dn_gelu(z);
  // z sigmoid(s): s = z, and (1 + tanh u) / 2 = sigmoid(2 u) for gelu's approximation
  if (act == CCQ_ACT_SILU) return z * dn_rcp(1.f + dn_exp(-z));
  if (act == CCQ_ACT_GELU_TANH) return z * dn_rcp(1.f + dn_exp(-1.595769122f * fmaf(0.044715f * z * z, z, z)));
  return z;
}

__device__ __forceinline__ float dn_value(int dt, const void* p, int64_t i) {
  if (dt == CCQ_F32) return reinterpret_cast<const float*>(p)[i];
  const uint32_t u = reinterpret_cast<const uint16_t*>(p)[i];
  return dt == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
}
// the n <= 4 values from i on
__device__ __forceinline__ f32x4 dn_load4(int dt, const void* p, int64_t i, int n) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (n < 4) {
    for (int e = 0; e < 3; ++e)
      if (e < n) v[e] = dn_value(dt, p, i + e);
  } else if (dt == CCQ_F32) {
    __builtin_memcpy(&v, reinterpret_cast<const float*>(p) + i, 16);
  } else {
    u32x2 b;
    __builtin_memcpy(&b, reinterpret_cast<const uint16_t*>(p) + i, 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = (b[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
      v[e] = dt == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
    }
  }
  return v;
}
__device__ __forceinline__ void dn_store4(int dt, void* p, int64_t i, int n, f32x4 v) {
  if (dt == CCQ_F32) {
    float* y = reinterpret_cast<float*>(p) + i;
    if (n >= 4) {
      __builtin_memcpy(y, &v, 16);
    } else {
      for (int e = 0; e < 3; ++e)
        if (e < n) y[e] = v[e];
    }
    return;
  }
  uint16_t* y = reinterpret_cast<uint16_t*>(p) + i;
  u32x2 b;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    b[e] = dt == CCQ_BF16 ? bf16x2_bits(v[2 * e], v[2 * e + 1])
                          : f32_to_f16_bits(v[2 * e]) | f32_to_f16_bits(v[2 * e + 1]) << 16;
  if (n >= 4) {
    __builtin_memcpy(y, &b, 8);
  } else {
    for (int e = 0; e < 3; ++e)
      if (e < n) y[e] = (uint16_t)(b[e >> 1] >> (16 * (e & 1)));
  }
}

// Four columns of y from column n on, of row `row`, from sums g (and u, the up
// half of a gated pair); e: the rows' expert.
__device__ __forceinline__ void dn_finish(const DenseP& p, int64_t row, int e, int n, f32x4 g, f32x4 u) {
  const int left = p.N - n;
  if (left <= 0) return;
  if (p.bias != nullptr) {
    const int64_t at = (int64_t)e * p.W + n;
    g += dn_load4(p.bias_dtype, p.bias, at, left);
    if (p.gated) u += dn_load4(p.bias_dtype, p.bias, at + p.N, left);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) g[i] = dn_act(p.act, g[i]);
  if (p.gated) g *= u;
  if (p.residual != nullptr) g += dn_load4(p.y_dtype, p.residual, row * p.ldr + n, left);
  dn_store4(p.y_dtype, p.y, row * p.ldy + n, left, g);
}

// ------------------------------------------------------- groups of rows --
// Row tile `tile` of BM rows of the experts' groups one behind the other, each
// padded to whole tiles, and behind them the rows of no expert (expert E).
// pick(tiles) is called with their number and gives the tile.  Every wave
// finds out by itself: lane l counts the experts from l PER on.
struct DnTile {
  int expert;      // E: rows of no expert; -1: no such tile
  int64_t row;     // first row
  int rows;
};

__device__ __forceinline__ int64_t dn_offset(const DenseP& p, int e) {
  return e > p.E ? p.M : imin64(p.M, e < 0 ? 0 : p.offsets[e] < 0 ? 0 : (int64_t)p.offsets[e]);
}
template <int BM, class Pick>
__device__ __forceinline__ DnTile dn_find_tile(const DenseP& p, Pick pick) {
  const int lane = lane_id();
  const int per = (p.E + 64) / 64, e0 = lane * per;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int e = e0 + i;
    if (e > p.E) break;
    const int64_t rows = dn_offset(p, e + 1) - dn_offset(p, e);
    if (rows > 0) mine += (int)((rows + BM - 1) / BM);
  }
  int upto = mine;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(upto, m, 64);
    upto += lane >= m ? o : 0;
  }
  const int total = __builtin_amdgcn_readlane(upto, 63);
  const int tile = pick(total);
  DnTile t = {-1, 0, 0};
  if (tile < 0 || tile >= total) return t;
  const uint64_t has = __ballot(tile < upto);
  const int l = __builtin_ctzll(has);  // the first lane whose experts reach the tile
  int at = tile - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
  for (int i = 0; i < per; ++i) {
    const int e = l * per + i;
    if (e > p.E) break;
    const int64_t first = dn_offset(p, e), rows = dn_offset(p, e + 1) - first;
    const int n = rows > 0 ? (int)((rows + BM - 1) / BM) : 0;
    if (at < n) {
      t.expert = e;
      t.row = first + (int64_t)at * BM;
      t.rows = (int)imin64(BM, rows - (int64_t)at * BM);
      return t;
    }
    at -= n;
  }
  return t;
}

// zeros into the rows of no expert, columns n0 .. n0 + BN - 1
__device__ __forceinline__ void dn_zero(const DenseP& p, const DnTile& t, int n0, int columns, int threads) {
  const int quads = columns / 4;
  for (int i = threadIdx.x; i < t.rows * quads; i += threads) {
    const int n = n0 + i % quads * 4;
    if (n < p.N) dn_store4(p.y_dtype, p.y, (t.row + i / quads) * p.ldy + n, p.N - n, f32x4{0.f, 0.f, 0.f, 0.f});
  }
}

// 8 values of a row from k on, at any element alignment; those from K on are 0.
// WHOLE: K is a multiple of 8, so either all or none are.
template <bool WHOLE>
__device__ __forceinline__ u32x4 dn_load8(const uint16_t* row, int k, int K) {
  u32x4 v = {0, 0, 0, 0};
  if (k + 8 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (k + e < K) v[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
  }
  return v;
}

// ------------------------------------------------------------- few rows --
// A workgroup takes NF groups of 16 rows of w and up to 16 MT rows of x; its 8
// waves take 32 U columns of K in turn, each multiplying what it loads, and
// their sums are added at the end in the waves' order.  w is read once, straight
// into the operand's registers: lane l holds 8 values of row l % 16 from column
// 8 (l / 16) on, so 4 neighbouring loads of a wave fill whole lines.
constexpr int FEW_WAVES = 8, FEW_THREADS = 64 * FEW_WAVES;

template <int DT, int MT, int NF, int U, bool WHOLE>
__global__ __launch_bounds__(FEW_THREADS) void dense_few_kernel(const DenseP p) {
  using Vec = typename DnVec<DT>::type;
  constexpr int BM = 16 * MT;
  __shared__ f32x4 sums[FEW_WAVES][MT * NF][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, k8 = (lane >> 4) * 8;
  DnTile t;
  int nt;
  if (p.offsets != nullptr) {
    nt = blockIdx.x % p.ntiles;
    t = dn_find_tile<BM>(p, [&](int) { return (int)blockIdx.x / p.ntiles; });
    if (t.expert < 0) return;
  } else {
    nt = blockIdx.x % p.ntiles;
    const int mt = blockIdx.x / p.ntiles;
    t = DnTile{0, (int64_t)mt * BM, (int)imin64(BM, p.M - (int64_t)mt * BM)};
  }
  const int columns = p.gated ? 8 * NF : 16 * NF, n0 = nt * columns;
  if (t.expert == p.E) {
    dn_zero(p, t, n0, columns, FEW_THREADS);
    return;
  }
  const uint16_t* w[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int n = p.gated ? n0 + f / 2 * 16 + r : n0 + f * 16 + r;
    const int64_t row = (int64_t)min(n, p.N - 1) + (p.gated && f & 1 ? p.N : 0);
    w[f] = reinterpret_cast<const uint16_t*>(p.w) + ((int64_t)t.expert * p.W + row) * p.K;
  }
  const uint16_t* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    x[m] = reinterpret_cast<const uint16_t*>(p.x) + (t.row + min(16 * m + r, t.rows - 1)) * p.ldx;
  f32x4 acc[NF][MT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[f][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int STEP = 32 * U;
  for (int k0 = wave * STEP; k0 < p.K; k0 += FEW_WAVES * STEP) {
    u32x4 wv[NF][U], xv[MT][U];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int u = 0; u < U; ++u) wv[f][u] = dn_load8<WHOLE>(w[f], k0 + 32 * u + k8, p.K);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < U; ++u) xv[m][u] = dn_load8<WHOLE>(x[m], k0 + 32 * u + k8, p.K);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[f][m] = dn_mfma(__builtin_bit_cast(Vec, wv[f][u]), __builtin_bit_cast(Vec, xv[m][u]), acc[f][m]);
  }
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave][f * MT + m][lane] = acc[f][m];
  __syncthreads();
  // a pair of groups (gated: gate and up) and 16 rows at a time
  const int groups = p.gated ? NF / 2 : NF;
  for (int i = threadIdx.x; i < groups * MT * 64; i += FEW_THREADS) {
    const int l = i & 63, m = i / 64 % MT, f = i / (64 * MT);
    const int fg = p.gated ? 2 * f : f;
    f32x4 g = sums[0][fg * MT + m][l], u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 1; v < FEW_WAVES; ++v) g += sums[v][fg * MT + m][l];
    if (p.gated) {
      u = sums[0][(fg + 1) * MT + m][l];
#pragma unroll
      for (int v = 1; v < FEW_WAVES; ++v) u += sums[v][(fg + 1) * MT + m][l];
    }
    const int row = 16 * m + (l & 15);
    if (row < t.rows) dn_finish(p, t.row + row, t.expert, n0 + f * 16 + 4 * (l >> 4), g, u);
  }
}

// ---------------------------------------------------------------- tiles --
// BM rows of x by BN rows of w (gated: 16 of the gate's and 16 of the up half's in
// turn), 64 columns of K a stage.  Rows in LDS are 128 bytes, their eight 16-byte
// pieces XORed with the row's low bits, so that the lanes which one cycle of an
// operand's read serves lie in different banks (no conflicts in the counters).
constexpr int DN_BK = 64;

struct DnPlace {  // a workgroup's tile
  DnTile t;
  int n0;         // first column
  int split;
};

// The tile of this workgroup: neighbouring tiles on one XCD, eight row tiles side
// by side, so that its workgroups share rows of both operands in its L2.
template <int BM>
__device__ __forceinline__ DnPlace dn_place(const DenseP& p, int columns) {
  DnPlace w = {};
  if (p.offsets != nullptr) {
    int at = 0;
    w.t = dn_find_tile<BM>(p, [&](int total) {
      const int all = total * p.ntiles;
      if ((int)blockIdx.x >= all) return -1;
      at = xcd_remap(blockIdx.x, all);
      return at / p.ntiles;
    });
    w.n0 = at % p.ntiles * columns;
    return w;
  }
  const int tiles = p.mtiles * p.ntiles, id = xcd_remap(blockIdx.x, tiles * p.splits);
  w.split = id / tiles;
  const int at = id % tiles, band = at / (8 * p.ntiles), inside = at % (8 * p.ntiles);
  const int high = min(8, p.mtiles - 8 * band), mt = 8 * band + inside % high;
  w.n0 = inside / high * columns;
  w.t = DnTile{0, (int64_t)mt * BM, (int)imin64(BM, p.M - (int64_t)mt * BM)};
  return w;
}

// row `q` of a tile's rows of w, as a row of w from row n0 on
__device__ __forceinline__ int64_t dn_wrow(const DenseP& p, int n0, int q) {
  const int n = p.gated ? (q >> 5) * 16 + (q & 15) : q;
  return (int64_t)min(n, p.N - 1 - n0) + (p.gated && q & 16 ? p.N : 0);
}

// The sums of a wave's FN x FM groups to y, or to the splits' sums: group (i, j)
// holds rows w0 + 16 i .. of the tile's w and row m0 + 16 j + lane % 16 of its x.
// They go through the wave's own piece of LDS, 16 rows at a time, so that rows of y
// are read and written in whole lines and the epilogue's code stands here once a
// group of rows (in place it took the accumulators' registers).
template <int FN>
constexpr int kScratch = 16 * (4 * FN + 1) * 16;  // bytes; a row's 4 FN quads and one, so that 16 rows start in 16 banks
template <int FM, int FN>
__device__ __forceinline__ void dn_write(const DenseP& p, const DnPlace& w, int m0, int w0, const f32x4 (&acc)[FN][FM],
                                         char* scratch) {
  constexpr int LINE = 4 * FN + 1;
  const int lane = lane_id();
  f32x4* own = reinterpret_cast<f32x4*>(scratch);
  const bool paired = p.gated && p.part == nullptr;
  const int quads = paired ? 2 * FN : 4 * FN;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
#pragma unroll
    for (int i = 0; i < FN; ++i) own[(lane & 15) * LINE + 4 * i + (lane >> 4)] = acc[i][j];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
    for (int at = lane; at < 16 * quads; at += 64) {
      const int r = at / quads, c = at - r * quads, row = m0 + 16 * j + r;
      if (row >= w.t.rows) break;
      if (paired) {
        const f32x4* q = own + r * LINE + (c & 3) + 8 * (c >> 2);
        dn_finish(p, w.t.row + row, w.t.expert, w.n0 + w0 / 2 + 4 * c, q[0], q[4]);
      } else if (p.part == nullptr) {
        dn_finish(p, w.t.row + row, w.t.expert, w.n0 + w0 + 4 * c, own[r * LINE + c], f32x4{0.f, 0.f, 0.f, 0.f});
      } else {
        const int q = w0 + 4 * c, n = w.n0 + (p.gated ? (q >> 5) * 16 + (q & 15) : q);
        if (n < p.N)
          dn_store4(CCQ_F32, p.part, ((int64_t)w.split * p.M + w.t.row + row) * p.W + n + (p.gated && q & 16 ? p.N : 0),
                    p.N - n, own[r * LINE + c]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// x and w aligned to 16 bytes in every row.  A stage's x and w are a unit each in
// a ring of five units of LDS, copied there by the loads themselves.  A stage is
// multiplied in two halves of 32 columns; each half's operands are read from LDS
// while the half before is multiplied, so the one barrier of a stage stands
// between its halves: behind it, all of this stage is in registers, its two units
// are free, and the next stage is in LDS.  Copies are spread over the products
// (64 of them at once fill the address unit and hold up the waves that issue
// them): w of the stage after the next follows the barrier, its x, into the ring's
// fifth unit, the first half of the next stage, so x is two stages ahead.
// 256 x 256, 4096 x 14336 x 4096: 327 us, 1470 TFLOP/s; the matrix unit is busy in
// 76 % of the cycles, at 1.75 GHz of 2.4: power bounds it.  (Two whole stages, the
// copies at once: 423 us; spread: 344; 32x32x16 products: 347 us, fewer cycles at
// a lower clock.)
template <int DT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void dense_tile_kernel(const DenseP p) {
  using Vec = typename DnVec<DT>::type;
  constexpr int WAVES = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int UNIT = (BM > BN ? BM : BN) * 128;
  constexpr int LX = BM / (8 * WAVES), LW = (BN + 8 * WAVES - 1) / (8 * WAVES);  // copies of a wave: 8 rows each
  constexpr int NM = FM * FN, NR = FM + FN;                                      // products and reads of a half
  static_assert(TM % 16 == 0 && TN % 16 == 0 && BM % (8 * WAVES) == 0 && 8 * WAVES * LW * 128 <= UNIT, "whole units");
  static_assert(NM >= 2 * NR && NM >= 4 * LW, "reads and copies fit between the products");
  __shared__ __align__(16) char lds[5 * UNIT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int columns = p.gated ? BN / 2 : BN;
  const DnPlace w = dn_place<BM>(p, columns);
  if (w.t.expert < 0) return;
  if (w.t.expert == p.E) {
    dn_zero(p, w.t, w.n0, columns, 64 * WAVES);
    return;
  }
  const int kfrom = w.split * p.kchunk, kto = min(p.K, kfrom + p.kchunk);
  const int stages = (kto - kfrom + DN_BK - 1) / DN_BK, whole = (kto - kfrom) / DN_BK;
  const uint16_t* xb = reinterpret_cast<const uint16_t*>(p.x) + w.t.row * p.ldx + kfrom;
  const uint16_t* wb = reinterpret_cast<const uint16_t*>(p.w) + ((int64_t)w.t.expert * p.W + w.n0) * p.K + kfrom;

  // copy i of a wave: rows 8 (wave + WAVES i) + lane / 8 of the unit, LDS piece lane % 8
  const int piece = (lane & 7) ^ (lane >> 3);  // its columns 8 piece .. + 7 (the row's low bits are lane / 8)
  uint32_t xo[LX], wo[LW];                     // in bytes, from xb and wb (rows past the tile's: its last one again)
#pragma unroll
  for (int i = 0; i < LX; ++i)
    xo[i] = (uint32_t)(2 * (min(8 * (wave + WAVES * i) + (lane >> 3), w.t.rows - 1) * p.ldx + 8 * piece));
#pragma unroll
  for (int i = 0; i < LW; ++i)
    wo[i] = (uint32_t)(2 * (dn_wrow(p, w.n0, min(8 * (wave + WAVES * i) + (lane >> 3), BN - 1)) * p.K + 8 * piece));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(&lds[0])) + wave * 1024;
  auto copy_x = [&](int i, int s, int unit) { dma16(xb + s * DN_BK, xo[i], lds0 + unit + i * WAVES * 1024); };
  auto copy_w = [&](int i, int s, int unit) { dma16(wb + s * DN_BK, wo[i], lds0 + unit + i * WAVES * 1024); };
  // the last stage, where K ends inside it: zeros from there on, in both operands
  const bool valid = (stages - 1) * DN_BK + 8 * piece < kto - kfrom;
  auto zero = [&](int i, int unit) {
    *reinterpret_cast<u32x4*>(&lds[unit + (wave + i * WAVES) * 1024 + lane * 16]) = u32x4{0, 0, 0, 0};
  };
  auto last_x = [&](int i, int unit) {
    if (valid) copy_x(i, stages - 1, unit);
    else zero(i, unit);
  };
  auto last_w = [&](int i, int unit) {
    if (valid) copy_w(i, stages - 1, unit);
    else zero(i, unit);
  };

  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Half {
    Vec x[FM], w[FN];
  };
  Half even, odd;  // operands of a stage's first and second 32 columns
  const int m0 = wave / WN * TM, w0 = wave % WN * TN;
  const uint32_t swz = ((lane >> 4) ^ (lane & 7)) * 16;  // of the first 32 columns; the others': ^ 64
  const uint32_t xat = (m0 + (lane & 15)) * 128 + swz, wat = (w0 + (lane & 15)) * 128 + swz;
  auto read = [&](Half& h, int r, uint32_t xa, uint32_t wa) {  // in the order in which the products take them
    if (r == 0)
      h.w[0] = *reinterpret_cast<const Vec*>(&lds[wa]);
    else if (r <= FM)
      h.x[r - 1] = *reinterpret_cast<const Vec*>(&lds[xa + (r - 1) * 2048]);
    else
      h.w[r - FM] = *reinterpret_cast<const Vec*>(&lds[wa + (r - FM) * 2048]);
  };
  auto ring = [](int u) { return u >= 5 * UNIT ? u - 5 * UNIT : u; };
  int ux = 0;  // the unit of this stage's x; its w is in the next one, the next stage in the two after that
  // COPY: of stage s + 2, 1 whole, 2 the last one; NEXT: there is a stage s + 1
  auto stage = [&](auto copy, auto next, int s) {
    constexpr int COPY = decltype(copy)::value;
    constexpr bool NEXT = decltype(next)::value;
    const int uw = ring(ux + UNIT), nx = ring(ux + 2 * UNIT), nw = ring(ux + 3 * UNIT), free = ring(ux + 4 * UNIT);
    {
      const uint32_t xa = (xat + ux) ^ 64, wa = (wat + uw) ^ 64;
#pragma unroll
      for (int q = 0; q < NM; ++q) {
        if (q % 2 == 0 && q / 2 < NR) read(odd, q / 2, xa, wa);
        if (COPY && q % (NM / LX) == NM / LX / 2) {
          if constexpr (COPY == 1) copy_x(q / (NM / LX), s + 2, free);
          else last_x(q / (NM / LX), free);
        }
        __builtin_amdgcn_sched_barrier(0);
        acc[q / FM][q % FM] = dn_mfma(even.w[q / FM], even.x[q % FM], acc[q / FM][q % FM]);
      }
    }
    if constexpr (NEXT) {
      wait_vmcnt<COPY == 1 ? LX : 0>();  // all but the copies just issued
      lds_barrier();
    }
#pragma unroll
    for (int q = 0; q < NM; ++q) {
      if (NEXT && q % 2 == 0 && q / 2 < NR) read(even, q / 2, xat + nx, wat + nw);
      if (COPY && q % 2 == 0 && q / 2 < LW) {
        if constexpr (COPY == 1) copy_w(q / 2, s + 2, ux);
        else last_w(q / 2, ux);
      }
      __builtin_amdgcn_sched_barrier(0);
      acc[q / FM][q % FM] = dn_mfma(odd.w[q / FM], odd.x[q % FM], acc[q / FM][q % FM]);
    }
    ux = nx;
  };
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    if (b < whole) {
#pragma unroll
      for (int i = 0; i < LX; ++i) copy_x(i, b, 2 * b * UNIT);
#pragma unroll
      for (int i = 0; i < LW; ++i) copy_w(i, b, (2 * b + 1) * UNIT);
    } else if (b < stages) {
#pragma unroll
      for (int i = 0; i < LX; ++i) last_x(i, 2 * b * UNIT);
#pragma unroll
      for (int i = 0; i < LW; ++i) last_w(i, (2 * b + 1) * UNIT);
    }
  }
  if (whole >= 2) wait_vmcnt<LX + LW>();
  else wait_vmcnt<0>();
  lds_barrier();
#pragma unroll
  for (int r = 0; r < NR; ++r) read(even, r, xat, wat + UNIT);
  constexpr std::integral_constant<int, 0> none{};
  constexpr std::integral_constant<int, 1> full{};
  constexpr std::integral_constant<int, 2> end{};
  int s = 0;
  for (; s + 2 < whole; ++s) stage(full, std::true_type{}, s);
  if (s + 2 < stages) stage(end, std::true_type{}, s++);
  if (s + 1 < stages) stage(none, std::true_type{}, s++);
  stage(none, std::false_type{}, s);
  __syncthreads();  // (the waves' scratch lies in the ring)
  dn_write<FM, FN>(p, w, m0, w0, acc, &lds[wave * kScratch<FN>]);
}

// The same product for rows at any alignment: stages pass through registers, two
// of them in LDS.
template <int DT>
__global__ __launch_bounds__(256, 2) void dense_ragged_kernel(const DenseP p) {
  using Vec = typename DnVec<DT>::type;
  constexpr int B = 128, WAVES = 4, FM = 4, FN = 4, LOADS = B / 8 / WAVES, UNIT = B * 128;
  __shared__ __align__(16) char lds[2][2 * UNIT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int columns = p.gated ? B / 2 : B;
  const DnPlace w = dn_place<B>(p, columns);
  if (w.t.expert < 0) return;
  if (w.t.expert == p.E) {
    dn_zero(p, w.t, w.n0, columns, 64 * WAVES);
    return;
  }
  const int kfrom = w.split * p.kchunk, kto = min(p.K, kfrom + p.kchunk);
  const int stages = (kto - kfrom + DN_BK - 1) / DN_BK;
  const int piece = (lane & 7) ^ (lane >> 3);
  const uint16_t *x[LOADS], *wr[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = 8 * (wave + WAVES * i) + (lane >> 3);
    x[i] = reinterpret_cast<const uint16_t*>(p.x) + (w.t.row + min(row, w.t.rows - 1)) * p.ldx;
    wr[i] = reinterpret_cast<const uint16_t*>(p.w) +
            ((int64_t)w.t.expert * p.W + w.n0 + dn_wrow(p, w.n0, row)) * p.K;
  }
  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int m0 = wave / 2 * 64, w0 = wave % 2 * 64;
  const uint32_t swz = ((lane >> 4) ^ (lane & 7)) * 16;
  const uint32_t xat = (m0 + (lane & 15)) * 128 + swz, wat = UNIT + (w0 + (lane & 15)) * 128 + swz;
  u32x4 xv[LOADS], wv[LOADS];
  auto load = [&](int s) {
    const int k = kfrom + s * DN_BK + 8 * piece;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      xv[i] = dn_load8<false>(x[i], k, kto);
      wv[i] = dn_load8<false>(wr[i], k, kto);
    }
  };
  load(0);
  for (int s = 0; s < stages; ++s) {
    char* to = &lds[s & 1][wave * 1024 + lane * 16];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      *reinterpret_cast<u32x4*>(to + i * WAVES * 1024) = xv[i];
      *reinterpret_cast<u32x4*>(to + UNIT + i * WAVES * 1024) = wv[i];
    }
    __syncthreads();
    if (s + 1 < stages) load(s + 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Vec xf[FM], wf[FN];
#pragma unroll
      for (int j = 0; j < FM; ++j) xf[j] = *reinterpret_cast<const Vec*>(&lds[s & 1][(xat ^ (64 * h)) + j * 2048]);
#pragma unroll
      for (int i = 0; i < FN; ++i) wf[i] = *reinterpret_cast<const Vec*>(&lds[s & 1][(wat ^ (64 * h)) + i * 2048]);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = dn_mfma(wf[i], xf[j], acc[i][j]);
    }
  }
  __syncthreads();
  dn_write<FM, FN>(p, w, m0, w0, acc, &lds[0][wave * kScratch<FN>]);
}

// The splits' sums added in order, and the epilogue.
__global__ __launch_bounds__(256) void dense_join_kernel(const DenseP p) {
  const int quads = (p.N + 3) / 4;
  const int64_t total = p.M * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / quads;
    const int n = (int)(i % quads) * 4;
    f32x4 g = {0.f, 0.f, 0.f, 0.f}, u = g;
    for (int s = 0; s < p.splits; ++s) {
      const float* part = p.part + ((int64_t)s * p.M + row) * p.W;
      g += dn_load4(CCQ_F32, part, n, p.N - n);
      if (p.gated) u += dn_load4(CCQ_F32, part, n + p.N, p.N - n);
    }
    dn_finish(p, row, 0, n, g, u);
  }
}

// ------------------------------------------------------------- dispatch --
constexpr int64_t FEW_ROWS = 64;

struct Plan {
  bool few, dma;
  int bm, bn;       // of the tile, or 16 MT and 16 NF
  int splits, kchunk;
};

// rows: of the batch, or of a group on average
Plan make_plan(const DenseP& p, int64_t rows, bool dma) {
  Plan q = {};
  q.few = rows <= FEW_ROWS;
  q.dma = dma;
  q.splits = 1;
  q.kchunk = p.K;
  if (q.few) {
    q.bm = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    q.bn = q.bm == 64 ? 64 : 32;
    return q;
  }
  const int64_t big = cdiv(p.M, 256) * cdiv(p.W, 256);
  if (dma && rows > 128 && big >= 192) {
    q.bm = q.bn = 256;
    return q;
  }
  q.bm = q.bn = 128;
  const int64_t tiles = cdiv(p.M, 128) * cdiv(p.W, 128);
  if (p.offsets == nullptr && tiles < 256) {
    const int64_t stages = cdiv(p.K, DN_BK);
    int64_t s = std::min<int64_t>(std::min<int64_t>(cdiv(512, tiles), stages / 8), 16);
    if (s > 1) {
      q.kchunk = (int)(cdiv(stages, s) * DN_BK);
      q.splits = (int)cdiv(p.K, q.kchunk);
    }
  }
  return q;
}

template <int DT, int MT, int NF, int U>
void launch_few(const DenseP& p, hipStream_t st) {
  const dim3 grid((uint32_t)((int64_t)p.mtiles * p.ntiles));
  if (p.K % 8 == 0)
    launch(dense_few_kernel<DT, MT, NF, U, true>, grid, dim3(FEW_THREADS), 0, st, p);
  else
    launch(dense_few_kernel<DT, MT, NF, U, false>, grid, dim3(FEW_THREADS), 0, st, p);
}

template <int DT>
int launch_dense(DenseP p, const Plan& q, hipStream_t st, const char* what) {
  const int columns = p.gated ? q.bn / 2 : q.bn;
  p.ntiles = (int)cdiv(p.N, columns);
  p.mtiles = (int)(p.offsets == nullptr ? cdiv(p.M, q.bm) : imin64(p.M, p.E + 1) + p.M / q.bm);
  p.splits = q.splits;
  p.kchunk = q.kchunk;
  const int64_t grid = (int64_t)p.mtiles * p.ntiles * q.splits;
  CCQ_REQUIRE(grid < 1 << 22, "%s: %lld tiles, too many for one launch", what, (long long)grid);
  if (q.few) {
    if (q.bm == 16)
      launch_few<DT, 1, 2, 4>(p, st);
    else if (q.bm == 32)
      launch_few<DT, 2, 2, 4>(p, st);
    else
      launch_few<DT, 4, 4, 2>(p, st);
    return launch_status(what);
  }
  if (q.bm == 256)
    launch(dense_tile_kernel<DT, 256, 256, 4, 2>, dim3((uint32_t)grid), dim3(512), 0, st, p);
  else if (q.dma)
    launch(dense_tile_kernel<DT, 128, 128, 2, 2>, dim3((uint32_t)grid), dim3(256), 0, st, p);
  else
    launch(dense_ragged_kernel<DT>, dim3((uint32_t)grid), dim3(256), 0, st, p);
  if (int rc = launch_status(what)) return rc;
  if (p.part != nullptr) {
    launch(dense_join_kernel, dim3((uint32_t)grid_for(p.M * cdiv(p.N, 4), 256)), dim3(256), 0, st, p);
    return launch_status(what);
  }
  return 0;
}

int check_dense(const char* what, const ccq_dense_args& a, bool grouped) {
  CCQ_REQUIRE(a.dtype == CCQ_F16 || a.dtype == CCQ_BF16, "%s: dtype %d, f16 or bf16", what, a.dtype);
  CCQ_REQUIRE(a.y_dtype >= 0 && a.y_dtype <= CCQ_BF16, "%s: y_dtype %d", what, a.y_dtype);
  CCQ_REQUIRE(a.bias == nullptr || (a.bias_dtype >= 0 && a.bias_dtype <= CCQ_BF16), "%s: bias_dtype %d", what,
              a.bias_dtype);
  CCQ_REQUIRE(a.act >= CCQ_ACT_NONE && a.act <= CCQ_ACT_SILU, "%s: act %d", what, a.act);
  CCQ_REQUIRE(a.M >= 0 && a.M <= 1 << 20, "%s: M=%lld rows, 0 to 2^20", what, (long long)a.M);
  CCQ_REQUIRE(a.K >= 1 && a.K <= 1 << 20 && a.N >= 1 && a.N <= 1 << 20, "%s: K=%lld, N=%lld, 1 to 2^20", what,
              (long long)a.K, (long long)a.N);
  CCQ_REQUIRE(a.M <= 1 || (a.ldx >= a.K && a.ldy >= a.N && (a.residual == nullptr || a.ldr >= a.N)),
              "%s: a row stride is shorter than its row", what);
  CCQ_REQUIRE(!grouped || (a.num_experts >= 1 && a.num_experts <= DN_MAX_E), "%s: num_experts=%lld, 1 to %lld", what,
              (long long)a.num_experts, (long long)DN_MAX_E);
  CCQ_REQUIRE(a.M == 0 || (a.x && a.w && a.y && (!grouped || a.offsets)), "%s: null pointer", what);
  const auto size = [](int dt) -> size_t { return dt == CCQ_F32 ? 4 : 2; };
  CCQ_REQUIRE(aligned(a.x, 2) && aligned(a.w, 2) && aligned(a.y, size(a.y_dtype)) &&
                  aligned(a.residual, size(a.y_dtype)) && aligned(a.bias, size(a.bias_dtype)) && aligned(a.offsets, 4),
              "%s: pointers must be aligned to their elements", what);
  return 0;
}

DenseP make_params(const ccq_dense_args& a, bool grouped) {
  DenseP p = {};
  p.x = a.x, p.w = a.w, p.bias = a.bias, p.residual = a.residual, p.y = a.y;
  p.offsets = grouped ? a.offsets : nullptr;
  p.ldx = a.ldx, p.ldr = a.ldr, p.ldy = a.ldy, p.M = a.M;
  p.K = (int)a.K, p.N = (int)a.N, p.W = (int)(a.gated ? 2 * a.N : a.N);
  p.E = grouped ? (int)a.num_experts : 1;  // (a batch's one "expert" is 0)
  p.gated = a.gated != 0, p.act = a.act, p.bias_dtype = a.bias_dtype, p.y_dtype = a.y_dtype;
  return p;
}

// LDS DMA: 16-byte pieces at 16-byte addresses, offsets from a tile's first row in 32 bits
bool can_dma(const ccq_dense_args& a) {
  const int64_t ldx = a.M > 1 ? a.ldx : a.K;
  return a.K % 8 == 0 && ldx % 8 == 0 && aligned(a.x, 16) && aligned(a.w, 16) && 256 * ldx + a.K < 1ll << 31 &&
         ((a.gated ? a.N : 0) + 256) * a.K < 1ll << 31;
}

Plan plan_of(const ccq_dense_args& a, const DenseP& p) {
  return make_plan(p, p.offsets != nullptr ? cdiv(a.M, a.num_experts) : a.M, can_dma(a));
}

int run_dense(const char* what, const ccq_dense_args& a, bool grouped) {
  if (int rc = check_dense(what, a, grouped)) return rc;
  if (a.M == 0) return 0;
  DenseP p = make_params(a, grouped);
  const Plan q = plan_of(a, p);
  if (q.splits > 1) {
    const size_t need = (size_t)q.splits * p.M * p.W * 4;
    CCQ_REQUIRE(a.workspace != nullptr && aligned(a.workspace, 16) && a.workspace_bytes >= need,
                "%s: workspace of %zu bytes needed", what, need);
    p.part = reinterpret_cast<float*>(a.workspace);
  }
  const hipStream_t st = as_stream(a.stream);
  return a.dtype == CCQ_BF16 ? launch_dense<CCQ_BF16>(p, q, st, what) : launch_dense<CCQ_F16>(p, q, st, what);
}

}  // namespace

}  // namespace ccq

using namespace ccq;

extern "C" size_t ccq_dense_linear_workspace_size(const ccq_dense_args* args) {
  if (args == nullptr || args->M < 1 || check_dense("ccq_dense_linear", *args, false)) return 0;
  const DenseP p = make_params(*args, false);
  const Plan q = plan_of(*args, p);
  return q.splits > 1 ? (size_t)q.splits * p.M * p.W * 4 : 0;
}

extern "C" int ccq_dense_linear(const ccq_dense_args* args) {
  CCQ_REQUIRE(args != nullptr, "ccq_dense_linear: null arguments");
  return run_dense("ccq_dense_linear", *args, false);
}

extern "C" int ccq_dense_linear_grouped(const ccq_dense_args* args) {
  CCQ_REQUIRE(args != nullptr, "ccq_dense_linear_grouped: null arguments");
  return run_dense("ccq_dense_linear_grouped", *args, true);
}
