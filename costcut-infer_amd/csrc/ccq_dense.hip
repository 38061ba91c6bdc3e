// Linears with weights of 16 bits and an epilogue, for a batch of rows and for
// rows grouped by expert:
//   z = x w^T + bias,   y = act(z) + residual,
//   gated (w holds 2N rows):   y = act(z[:, :N]) * z[:, N:] + residual,
// x [M, K], w [N, K] (grouped: w[e] for the rows offsets[e] .. offsets[e + 1] - 1),
// products and everything after them in float32, y rounded once.
//
// All kernels give the matrix instructions w as their first operand, so a lane
// ends with four neighbouring columns of one row of y, and with the gate and up
// rows of w in turn (16 by 16) also both halves of a gated value: the epilogue
// needs no exchange.
//
// dense_few_kernel   up to 16 rows: w goes from memory to registers, the waves of a
//                    workgroup share K and add up at the end.
// dense_mid_kernel   tiles of 32 rows, through a ring of stages in LDS.
// dense_tile_kernel  large tiles, the products interleaved with the next ones' reads.
// dense_ring_kernel  smaller ones, more stages on their way.
// dense_ragged_kernel  rows at any alignment.
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
  float* part;            // [splits][M][P] sums of K's splits, or null
  const int32_t* offsets; // grouped, or null
  int64_t ldx, ldr, ldy;
  int64_t M;              // rows in all
  int K, N, W;            // W: rows of w, N or 2N
  int half, P;            // columns of a row of part: N (gated: of each half), to whole quads, in all
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
// keep their relative accuracy, and it takes a third of erff's instructions.  The
// factors 1 / sqrt 2 and 1 / 2 are in the constants: 0.33 / sqrt 2, the coefficients'
// halves, log2(e) / 2.
__device__ __forceinline__ float dn_gelu(float z) {
  const float t = dn_rcp(fmaf(0.233345238f, fabsf(z), 1.f));
  float q = fmaf(t, -0.06767245f, 0.230116985f);
  q = fmaf(t, q, -0.17557224f);
  q = fmaf(t, q, 0.204247675f);
  q = fmaf(t, q, 0.023611515f);
  q = fmaf(t, q, 0.100611595f);
  q = fmaf(t, q, 0.091478025f);
  q = fmaf(t, q, 0.0931789f);
  q = q * t * __builtin_amdgcn_exp2f(z * z * -0.72134752f);
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

struct f32x8 {
  f32x4 lo, hi;
};
__device__ __forceinline__ f32x8 dn_floats8(int dt, u32x4 b) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = (b[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
    (e < 4 ? v.lo : v.hi)[e & 3] = dt == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
  }
  return v;
}
__device__ __forceinline__ u32x4 dn_bits8(int dt, const f32x8& v) {
  u32x4 b;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x4& h = e < 2 ? v.lo : v.hi;
    const float a = h[2 * (e & 1)], c = h[2 * (e & 1) + 1];
    b[e] = dt == CCQ_BF16 ? bf16x2_bits(a, c) : f32_to_f16_bits(a) | f32_to_f16_bits(c) << 16;
  }
  return b;
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
// pick(tiles) is called with their number and gives the tile.  Every wave finds it
// by itself, 256 experts at a time: lane l looks at the four experts l, l + 64, ..
struct DnTile {
  int expert;      // E: rows of no expert; -1: no such tile
  int64_t row;     // first row
  int rows;
};

template <int BM, class Pick>
__device__ __forceinline__ DnTile dn_find_tile(const DenseP& p, Pick pick) {
  constexpr int SETS = 4;
  const int lane = lane_id(), M = (int)p.M;
  int first[SETS], rows[SETS], tiles[SETS], upto[SETS], all[SETS];
  auto look = [&](int base) {
    int next[SETS];
#pragma unroll
    for (int c = 0; c < SETS; ++c) {  // (all of the loads at once)
      const int e = base + 64 * c + lane;
      first[c] = p.offsets[min(e, p.E)];
      next[c] = p.offsets[min(e + 1, p.E)];
    }
    int sum = 0;
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
      const int e = base + 64 * c + lane;
      first[c] = min(max(first[c], 0), M);
      rows[c] = e > p.E ? 0 : (e == p.E ? M : min(max(next[c], 0), M)) - first[c];
      tiles[c] = rows[c] > 0 ? (rows[c] + BM - 1) / BM : 0;
      upto[c] = wave_scan(tiles[c]);
      all[c] = __builtin_amdgcn_readlane(upto[c], 63);
      sum += all[c];
    }
    return sum;
  };
  int total = look(0);
  for (int base = 64 * SETS; base <= p.E; base += 64 * SETS) total += look(base);
  int at = pick(total);
  DnTile t = {-1, 0, 0};
  if (at < 0 || at >= total) return t;
  for (int base = 0; base <= p.E; base += 64 * SETS) {
    if (p.E >= 64 * SETS) look(base);
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
      if (t.expert < 0 && at < all[c]) {
        const int l = __builtin_ctzll(__ballot(at < upto[c]));  // the first lane whose experts reach the tile
        at -= __builtin_amdgcn_readlane(upto[c], l) - __builtin_amdgcn_readlane(tiles[c], l);
        t.expert = base + 64 * c + l;
        t.row = __builtin_amdgcn_readlane(first[c], l) + (int64_t)at * BM;
        t.rows = min(BM, __builtin_amdgcn_readlane(rows[c], l) - at * BM);
      }
      at -= all[c];
    }
    if (t.expert >= 0) break;
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
// A workgroup takes NF groups of 16 rows of w and up to 16 MT rows of x; its waves
// take 32 U columns of K in turn, each multiplying what it loads, and their sums
// are added at the end in the waves' order.  w is read once, straight into the
// operand's registers, the next columns while these are multiplied: lane l holds 8
// values of row l % 16 from column 8 (l / 16) on, so neighbouring loads of a wave
// fill whole lines.  M=1 K=2048 N=5632 7.2 us among others; M=16 K=4096 N=2x14336
// 48.9 us, 4.8 TB/s.
//
// Loads of 16 bytes at odd elements run at half the rate of those at dwords, so where
// rows start at odd ones (ROWS == ODD) their lanes load the dwords around their eight
// values: four from the one that holds the first, and the one that holds the last (a
// lane at an even element loads its own last dword again), moved by a value when they
// are multiplied.  A dword that holds a value of a row lies in the row's allocation.
// M=8 K=2049: N=8192 20.7 us by loads at odd elements, 11.1 by dwords (K=2050 10.7);
// N=20480 52 and 32.
enum Rows { WHOLE, EVEN, ODD };  // K in whole eights; rows from whole dwords on; any

template <int DT, int MT, int NF, int U, int WAVES, Rows ROWS>
__global__ __launch_bounds__(64 * WAVES) void dense_few_kernel(const DenseP p) {
  using Vec = typename DnVec<DT>::type;
  constexpr int BM = 16 * MT, THREADS = 64 * WAVES, STEP = 32 * U;
  __shared__ f32x4 sums[WAVES][MT * NF][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, k8 = (lane >> 4) * 8;
  const int nt = blockIdx.x % p.ntiles, mt = blockIdx.x / p.ntiles;
  DnTile t;
  if (p.offsets != nullptr) {
    t = dn_find_tile<BM>(p, [&](int) { return mt; });
    if (t.expert < 0) return;
  } else {
    t = DnTile{0, (int64_t)mt * BM, (int)imin64(BM, p.M - (int64_t)mt * BM)};
  }
  const int columns = p.gated ? 8 * NF : 16 * NF, n0 = nt * columns;
  if (t.expert == p.E) {
    dn_zero(p, t, n0, columns, THREADS);
    return;
  }
  const uint16_t* w[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int n = p.gated ? n0 + f / 2 * 16 + r : n0 + f * 16 + r;
    const int64_t row = (int64_t)min(n, p.N - 1) + (p.gated && f & 1 ? p.N : 0);
    w[f] = reinterpret_cast<const uint16_t*>(p.w) + ((int64_t)t.expert * p.W + row) * p.K + k8;
  }
  const uint16_t* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    x[m] = reinterpret_cast<const uint16_t*>(p.x) + (t.row + min(16 * m + r, t.rows - 1)) * p.ldx + k8;
  f32x4 acc[NF][MT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[f][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Pieces {
    u32x4 w[NF][U], x[MT][U];
  };
  struct OddPieces : Pieces {
    uint32_t wl[NF][U], xl[MT][U];  // the dwords of the last values
  };
  using Step = std::conditional_t<ROWS == ODD, OddPieces, Pieces>;
  const auto odd = [](const uint16_t* row) { return (uint32_t)(reinterpret_cast<uintptr_t>(row) >> 1) & 1; };
  auto load = [&](Step& s, int k0) {
    if constexpr (ROWS == ODD) {
      const auto full = [&](u32x4& v, uint32_t& last, const uint16_t* row, int k) {
        const uint32_t o = odd(row);
        __builtin_memcpy(&v, row + k - o, 16);
        __builtin_memcpy(&last, row + k + 6 + o, 4);
      };
      const auto tail = [&](u32x4& v, uint32_t& last, const uint16_t* row, int k) {
        v = dn_load8<false>(row, k, p.K - k8);
        last = v[3] >> 16;
        if (odd(row)) v = u32x4{v[0] << 16, v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16};
      };
      const auto all = [&](const auto& one) {
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
          for (int u = 0; u < U; ++u) one(s.w[f][u], s.wl[f][u], w[f], k0 + 32 * u);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int u = 0; u < U; ++u) one(s.x[m][u], s.xl[m][u], x[m], k0 + 32 * u);
      };
      if (k0 + STEP <= p.K) all(full);
      else all(tail);
    } else if (k0 + STEP <= p.K) {
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&s.w[f][u], w[f] + k0 + 32 * u, 16);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&s.x[m][u], x[m] + k0 + 32 * u, 16);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + 32 * u;
#pragma unroll
        for (int f = 0; f < NF; ++f) s.w[f][u] = dn_load8<ROWS == WHOLE>(w[f], k, p.K - k8);
#pragma unroll
        for (int m = 0; m < MT; ++m) s.x[m][u] = dn_load8<ROWS == WHOLE>(x[m], k, p.K - k8);
      }
    }
  };
  auto multiply = [&](const Step& s) {
    const auto value = [&](const u32x4& v, uint32_t last, const uint16_t* row) {
      const uint32_t by = 16 * odd(row);
      return __builtin_bit_cast(Vec, u32x4{__builtin_amdgcn_alignbit(v[1], v[0], by), __builtin_amdgcn_alignbit(v[2], v[1], by),
                                           __builtin_amdgcn_alignbit(v[3], v[2], by), __builtin_amdgcn_alignbit(last, v[3], by)});
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if constexpr (ROWS == ODD)
            acc[f][m] = dn_mfma(value(s.w[f][u], s.wl[f][u], w[f]), value(s.x[m][u], s.xl[m][u], x[m]), acc[f][m]);
          else
            acc[f][m] = dn_mfma(__builtin_bit_cast(Vec, s.w[f][u]), __builtin_bit_cast(Vec, s.x[m][u]), acc[f][m]);
        }
  };
  constexpr int STRIDE = WAVES * STEP;
  int k0 = wave * STEP;
  if (k0 < p.K) {
    Step a, b;
    load(a, k0);
    for (;;) {
      if ((k0 += STRIDE) >= p.K) {
        multiply(a);
        break;
      }
      load(b, k0);
      multiply(a);
      if ((k0 += STRIDE) >= p.K) {
        multiply(b);
        break;
      }
      load(a, k0);
      multiply(b);
    }
  }
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave][f * MT + m][lane] = acc[f][m];
  __syncthreads();
  // a pair of groups (gated: gate and up) and 16 rows at a time
  const int groups = p.gated ? NF / 2 : NF;
  for (int i = threadIdx.x; i < groups * MT * 64; i += THREADS) {
    const int l = i & 63, m = i / 64 % MT, f = i / (64 * MT);
    const int fg = p.gated ? 2 * f : f;
    f32x4 g = sums[0][fg * MT + m][l], u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 1; v < WAVES; ++v) g += sums[v][fg * MT + m][l];
    if (NF > 1 && p.gated) {
      u = sums[0][(fg + 1) * MT + m][l];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) u += sums[v][(fg + 1) * MT + m][l];
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

// Waits until at most `n` stages of L copies each are on their way (n >= N: N).
template <int N, int L>
__device__ __forceinline__ void wait_stages(int n) {
  if constexpr (N > 0) {
    if (n < N) {
      wait_stages<N - 1, L>(n);
      return;
    }
  }
  wait_vmcnt<N * L>();
}

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
// Bias, activation and gate are applied where the sums are; then 16 rows at a time
// go through the wave's own piece of LDS, so that y and the residual are accessed
// 16 bytes a lane in whole lines (8 bytes a lane in 16 rows at once take 4 to 7
// times as long: 14000 cycles of a 256 x 256 tile).
template <int FN>
constexpr int kScratch = 16 * (4 * FN + 1) * 16;  // bytes; a row's 4 FN quads and one, so that 16 rows start in 16 banks
constexpr int dn_pow2(int n) { return n <= 1 ? 1 : 2 * dn_pow2((n + 1) / 2); }

// row group j to the wave's LDS, behind what was read there before: every group of columns, or every second one
template <int FM, int FN, int EVERY>
__device__ __forceinline__ void dn_dump(const f32x4 (&acc)[FN][FM], f32x4* own, int j) {
  const int lane = lane_id();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int i = 0; i < FN; i += EVERY) own[(lane & 15) * (4 * (FN / EVERY) + 1) + 4 * (i / EVERY) + (lane >> 4)] = acc[i][j];
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

template <int FM, int FN>
__device__ __forceinline__ void dn_act_all(int act, int every, f32x4 (&acc)[FN][FM]) {
  auto all = [&](auto a) {
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if (i % 2 && every == 2) continue;  // (the up half's)
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = dn_act(decltype(a)::value, acc[i][j][e]);
    }
  };
  if (act == CCQ_ACT_SILU) all(std::integral_constant<int, CCQ_ACT_SILU>{});
  else if (act == CCQ_ACT_GELU) all(std::integral_constant<int, CCQ_ACT_GELU>{});
  else if (act == CCQ_ACT_GELU_TANH) all(std::integral_constant<int, CCQ_ACT_GELU_TANH>{});
  else if (act == CCQ_ACT_RELU) all(std::integral_constant<int, CCQ_ACT_RELU>{});
}

// y's rows from the wave's LDS; EVERY 2: the groups of columns that a gated product leaves
template <int FM, int FN, int EVERY>
__device__ __forceinline__ void dn_write_y(const DenseP& p, const DnPlace& w, int m0, int w0, const f32x4 (&acc)[FN][FM],
                                           f32x4* own) {
  constexpr int GROUPS = FN / EVERY, OCTS = 2 * GROUPS, SIDE = dn_pow2(OCTS), LINE = 4 * GROUPS + 1;
  constexpr int STEP = 64 / SIDE < 16 ? 64 / SIDE : 16, TURNS = 16 / STEP;  // rows of an access, accesses of 16 rows
  const int lane = lane_id(), c = lane & (SIDE - 1), r0 = lane / SIDE;
  const int n = w.n0 + w0 / EVERY + 8 * c;
  const int left = c < OCTS && r0 < 16 ? p.N - n : 0;
  const f32x4* from = own + (r0 & 15) * LINE + 2 * c;
  if (p.y_dtype != CCQ_F32 && (p.N % 8 == 0 || w.n0 + w0 / EVERY + 16 * GROUPS <= p.N)) {  // whole eights
    // the residual two row groups ahead: turns that wait for their own cost a tile 16 us
    constexpr int AHEAD = FM < 2 ? FM : 2;
    u32x4 res[AHEAD][TURNS];
    auto ask = [&](int j) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int row = m0 + 16 * j + r0 + i * STEP;
        if (row < w.t.rows && left > 0)
          __builtin_memcpy(&res[j % AHEAD][i], reinterpret_cast<const uint16_t*>(p.residual) + (w.t.row + row) * p.ldr + n, 16);
      }
    };
    auto rows = [&](auto residual) {
      constexpr bool RES = decltype(residual)::value;
      if constexpr (RES) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) ask(j);
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        dn_dump<FM, FN, EVERY>(acc, own, j);
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
          const int row = m0 + 16 * j + r0 + i * STEP;
          f32x8 v = {from[i * STEP * LINE], from[i * STEP * LINE + 1]};
          if constexpr (RES) {
            const f32x8 r = dn_floats8(p.y_dtype, res[j % AHEAD][i]);
            v.lo += r.lo;
            v.hi += r.hi;
          }
          const u32x4 bits = dn_bits8(p.y_dtype, v);
          if (row < w.t.rows && left > 0)
            __builtin_memcpy(reinterpret_cast<uint16_t*>(p.y) + (w.t.row + row) * p.ldy + n, &bits, 16);
        }
        if constexpr (RES) {
          if (j + AHEAD < FM) ask(j + AHEAD);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (p.residual != nullptr) rows(std::true_type{});
    else rows(std::false_type{});
    return;
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    dn_dump<FM, FN, EVERY>(acc, own, j);
#pragma unroll 1
    for (int i = 0; i < 2 * TURNS; ++i) {
      const int row = m0 + 16 * j + r0 + (i >> 1) * STEP, at = n + 4 * (i & 1), some = left - 4 * (i & 1);
      if (row >= w.t.rows || some <= 0) continue;
      f32x4 v = from[(i >> 1) * STEP * LINE + (i & 1)];
      if (p.residual != nullptr) v += dn_load4(p.y_dtype, p.residual, (w.t.row + row) * p.ldr + at, some);
      dn_store4(p.y_dtype, p.y, (w.t.row + row) * p.ldy + at, some, v);
    }
  }
}

template <int FM, int FN>
__device__ __forceinline__ void dn_write(const DenseP& p, const DnPlace& w, int m0, int w0, f32x4 (&acc)[FN][FM],
                                         char* scratch) {
  f32x4* own = reinterpret_cast<f32x4*>(scratch);
  const int lane = lane_id();
  if (p.part != nullptr) {
    constexpr int QUADS = 4 * FN, SIDE = dn_pow2(QUADS), STEP = 64 / SIDE;
    const int c = lane & (SIDE - 1), r0 = lane / SIDE, q = w0 + 4 * c;
    const int n = w.n0 + (p.gated ? (q >> 5) * 16 + (q & 15) : q);
    const bool own_columns = c < QUADS && n < p.half;
    float* part = p.part + ((int64_t)w.split * p.M + w.t.row) * p.P + n + (p.gated && q & 16 ? p.half : 0);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      dn_dump<FM, FN, 1>(acc, own, j);
#pragma unroll 2
      for (int r = r0; r < 16; r += STEP) {
        const int row = m0 + 16 * j + r;
        if (row < w.t.rows && own_columns)
          *reinterpret_cast<f32x4*>(part + (int64_t)row * p.P) = own[r * (4 * FN + 1) + c];
      }
    }
    return;
  }
  const int every = p.gated ? 2 : 1;
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const int q = w0 + 16 * i, n = w.n0 + (p.gated ? (q >> 5) * 16 : q) + 4 * (lane >> 4);
      if (n >= p.N) continue;
      const f32x4 b = dn_load4(p.bias_dtype, p.bias, (int64_t)w.t.expert * p.W + n + (p.gated && i % 2 ? p.N : 0), p.N - n);
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] += b;
    }
  }
  dn_act_all<FM, FN>(p.act, every, acc);
  if (!p.gated) {
    dn_write_y<FM, FN, 1>(p, w, m0, w0, acc, own);
  } else if constexpr (FN % 2 == 0) {
#pragma unroll
    for (int i = 0; i < FN; i += 2)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] *= acc[i + 1][j];
    dn_write_y<FM, FN, 2>(p, w, m0, w0, acc, own);
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
// 256 x 256, 4096 x 14336 x 4096: 327 to 332 us, 1470 TFLOP/s; the matrix unit is
// busy in 76 % of the cycles, and the clock falls to 1.75 GHz of 2.4 under this load.
// That is no limit of the card: a library's plain product of these sizes takes 294 to
// 308 us, for a reason that the counters do not name.  (Two whole stages, the copies at
// once: 423 us; spread: 344; 32x32x16 products: 347 us, fewer cycles at a lower clock.)
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
  constexpr std::integral_constant<int, 0> none{};
  constexpr std::integral_constant<int, 1> full{};
  constexpr std::integral_constant<int, 2> end{};
  int s = 0;
  if (m0 >= w.t.rows) {
    // a wave whose rows are all behind the tile's end only copies: the others of a short tile have the matrix units
    // to themselves
    for (; s + 1 < stages; ++s) {
      const int nx = ring(ux + 2 * UNIT), free = ring(ux + 4 * UNIT);
      if (s + 2 < whole)
#pragma unroll
        for (int i = 0; i < LX; ++i) copy_x(i, s + 2, free);
      else if (s + 2 < stages)
#pragma unroll
        for (int i = 0; i < LX; ++i) last_x(i, free);
      if (s + 2 < whole) wait_vmcnt<LX>();
      else wait_vmcnt<0>();
      lds_barrier();
      if (s + 2 < whole)
#pragma unroll
        for (int i = 0; i < LW; ++i) copy_w(i, s + 2, ux);
      else if (s + 2 < stages)
#pragma unroll
        for (int i = 0; i < LW; ++i) last_w(i, ux);
      ux = nx;
    }
    __syncthreads();
    return;
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) read(even, r, xat, wat + UNIT);
  for (; s + 2 < whole; ++s) stage(full, std::true_type{}, s);
  if (s + 2 < stages) stage(end, std::true_type{}, s++);
  if (s + 1 < stages) stage(none, std::true_type{}, s++);
  stage(none, std::false_type{}, s);
  __syncthreads();  // (the waves' scratch lies in the ring)
  dn_write<FM, FN>(p, w, m0, w0, acc, &lds[wave * kScratch<FN>]);
}

// Smaller tiles of the same form, with A whole stages on their way: they are
// multiplied in a fraction of the time that a stage takes from memory, and what
// counts is that every CU has one.  A stage's operands are read half by half while
// the half before is multiplied; the barrier stands between the halves as above.
// One workgroup a CU, K=4096: 64 x 64 0.31 us a stage, 128 x 128 0.41 to 0.47 (in the
// form above, which leaves room for two: 0.50 to 0.72), 256 x 128 0.7 to 0.9.
template <int DT, int BM, int BN, int WM, int WN, int A>
__global__ __launch_bounds__(64 * WM * WN, 2) void dense_ring_kernel(const DenseP p) {
  using Vec = typename DnVec<DT>::type;
  constexpr int WAVES = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int LX = BM / (8 * WAVES), LW = BN / (8 * WAVES), LOADS = LX + LW, STAGE = (BM + BN) * 128, D = A + 1;
  constexpr int NM = FM * FN, NR = FM + FN;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole copies");
  __shared__ __align__(16) char lds[D * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int columns = p.gated ? BN / 2 : BN;
  const DnPlace w = dn_place<BM>(p, columns);
  if (w.t.expert < 0) return;
  if (w.t.expert == p.E) {
    dn_zero(p, w.t, w.n0, columns, 64 * WAVES);
    return;
  }
  const int kfrom = w.split * p.kchunk, klen = min(p.K, kfrom + p.kchunk) - kfrom;
  const int stages = (klen + DN_BK - 1) / DN_BK, whole = klen / DN_BK;
  const uint16_t* xb = reinterpret_cast<const uint16_t*>(p.x) + w.t.row * p.ldx + kfrom;
  const uint16_t* wb = reinterpret_cast<const uint16_t*>(p.w) + ((int64_t)w.t.expert * p.W + w.n0) * p.K + kfrom;
  const int piece = (lane & 7) ^ (lane >> 3);
  uint32_t xo[LX], wo[LW];
#pragma unroll
  for (int i = 0; i < LX; ++i)
    xo[i] = (uint32_t)(2 * (min(8 * (wave + WAVES * i) + (lane >> 3), w.t.rows - 1) * p.ldx + 8 * piece));
#pragma unroll
  for (int i = 0; i < LW; ++i) wo[i] = (uint32_t)(2 * (dn_wrow(p, w.n0, 8 * (wave + WAVES * i) + (lane >> 3)) * p.K + 8 * piece));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(&lds[0])) + wave * 1024;
  auto copy = [&](int i, int s, int slot) {
    if (i < LW) dma16(wb + s * DN_BK, wo[i < LW ? i : 0], lds0 + slot + (BM / 8 + i * WAVES) * 1024);
    else dma16(xb + s * DN_BK, xo[i < LW ? 0 : i - LW], lds0 + slot + (i - LW) * WAVES * 1024);
  };
  auto copy_last = [&](int slot) {  // K ends inside: zeros from there on, in both operands
    const bool valid = (stages - 1) * DN_BK + 8 * piece < klen;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if (valid)
        copy(i, stages - 1, slot);
      else
        *reinterpret_cast<u32x4*>(&lds[slot + (wave + (i < LW ? BM / 8 + i * WAVES : (i - LW) * WAVES)) * 1024 + lane * 16]) =
            u32x4{0, 0, 0, 0};
    }
  };
  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Half {
    Vec x[FM], w[FN];
  };
  Half even, odd;
  const int m0 = wave / WN * TM, w0 = wave % WN * TN;
  const uint32_t swz = ((lane >> 4) ^ (lane & 7)) * 16;
  const uint32_t xat = (m0 + (lane & 15)) * 128 + swz, wat = (BM + w0 + (lane & 15)) * 128 + swz;
  auto read = [&](Half& h, int r, int slot, uint32_t half) {
    if (r == 0)
      h.w[0] = *reinterpret_cast<const Vec*>(&lds[slot + (wat ^ half)]);
    else if (r <= FM)
      h.x[r - 1] = *reinterpret_cast<const Vec*>(&lds[slot + (xat ^ half) + (r - 1) * 2048]);
    else
      h.w[r - FM] = *reinterpret_cast<const Vec*>(&lds[slot + (wat ^ half) + (r - FM) * 2048]);
  };
#pragma unroll
  for (int s = 0; s < D; ++s) {
    if (s < whole) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) copy(i, s, s * STAGE);
    } else if (s < stages) {
      copy_last(s * STAGE);
    }
  }
  if (stages >= D) wait_vmcnt<A * LOADS>();
  else wait_vmcnt<0>();
  lds_barrier();
#pragma unroll
  for (int r = 0; r < NR; ++r) read(even, r, 0, 0);
  int slot = 0;
  for (int s = 0; s < stages; ++s) {
    const int next = slot + STAGE == D * STAGE ? 0 : slot + STAGE;
#pragma unroll
    for (int q = 0; q < NM; ++q) {
#pragma unroll
      for (int r = q * NR / NM; r < (q + 1) * NR / NM; ++r) read(odd, r, slot, 64);
      __builtin_amdgcn_sched_barrier(0);
      acc[q / FM][q % FM] = dn_mfma(even.w[q / FM], even.x[q % FM], acc[q / FM][q % FM]);
    }
    if (s + A < stages) wait_vmcnt<(A - 1) * LOADS>();  // stage s + 1 is there; those behind it may be on their way
    else wait_vmcnt<0>();
    lds_barrier();
    const bool more = s + D < whole;
    if (!more && s + D < stages) copy_last(slot);
#pragma unroll
    for (int q = 0; q < NM; ++q) {
#pragma unroll
      for (int r = q * NR / NM; r < (q + 1) * NR / NM; ++r) read(even, r, next, 0);  // (behind the last stage: not used)
#pragma unroll
      for (int i = q * LOADS / NM; i < (q + 1) * LOADS / NM; ++i)
        if (more) copy(i, s + D, slot);
      __builtin_amdgcn_sched_barrier(0);
      acc[q / FM][q % FM] = dn_mfma(odd.w[q / FM], odd.x[q % FM], acc[q / FM][q % FM]);
    }
    slot = next;
  }
  __syncthreads();  // (the waves' scratch lies in the ring)
  dn_write<FM, FN>(p, w, m0, w0, acc, &lds[wave * kScratch<FN>]);
}

// 32 rows: w's way from memory bounds them, so a simple loop, K split over
// workgroups, and a ring of D stages that are on their way while one is multiplied.
// Four waves, 2 x 2.  64 experts of 6 rows, 1408 -> 2048: 68 us, 5.4 TB/s.
template <int DT, int BM, int BN, int D>
__global__ __launch_bounds__(256) void dense_mid_kernel(const DenseP p) {
  using Vec = typename DnVec<DT>::type;
  constexpr int WAVES = 4, TM = BM / 2, TN = BN / 2, FM = TM / 16, FN = TN / 16;
  constexpr int LX = BM / (8 * WAVES), LW = BN / (8 * WAVES), STAGE = (BM + BN) * 128;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole copies");
  __shared__ __align__(16) char lds[D * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int columns = p.gated ? BN / 2 : BN;
  const DnPlace w = dn_place<BM>(p, columns);
  if (w.t.expert < 0) return;
  if (w.t.expert == p.E) {
    dn_zero(p, w.t, w.n0, columns, 64 * WAVES);
    return;
  }
  const int kfrom = w.split * p.kchunk, kto = min(p.K, kfrom + p.kchunk);
  const int stages = (kto - kfrom + DN_BK - 1) / DN_BK;
  const uint16_t* xb = reinterpret_cast<const uint16_t*>(p.x) + w.t.row * p.ldx + kfrom;
  const uint16_t* wb = reinterpret_cast<const uint16_t*>(p.w) + ((int64_t)w.t.expert * p.W + w.n0) * p.K + kfrom;
  const int piece = (lane & 7) ^ (lane >> 3);
  uint32_t xo[LX], wo[LW];
#pragma unroll
  for (int i = 0; i < LX; ++i)
    xo[i] = (uint32_t)(2 * (min(8 * (wave + WAVES * i) + (lane >> 3), w.t.rows - 1) * p.ldx + 8 * piece));
#pragma unroll
  for (int i = 0; i < LW; ++i) wo[i] = (uint32_t)(2 * (dn_wrow(p, w.n0, 8 * (wave + WAVES * i) + (lane >> 3)) * p.K + 8 * piece));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(&lds[0])) + wave * 1024;
  auto copy = [&](int s, int slot) {
    const uint16_t *xs = xb + s * DN_BK, *ws = wb + s * DN_BK;
    const uint32_t to = lds0 + slot;
    if ((s + 1) * DN_BK <= kto - kfrom) {
#pragma unroll
      for (int i = 0; i < LW; ++i) dma16(ws, wo[i], to + (BM / 8 + i * WAVES) * 1024);
#pragma unroll
      for (int i = 0; i < LX; ++i) dma16(xs, xo[i], to + i * WAVES * 1024);
    } else {  // K ends inside: zeros from there on, in both operands (each copy has lanes before the end)
      const bool valid = s * DN_BK + 8 * piece < kto - kfrom;
#pragma unroll
      for (int i = 0; i < LX + LW; ++i) {
        const int at = i < LX ? i * WAVES : BM / 8 + (i - LX) * WAVES;
        if (valid) dma16(i < LX ? xs : ws, i < LX ? xo[i < LX ? i : 0] : wo[i < LX ? 0 : i - LX], to + at * 1024);
        else *reinterpret_cast<u32x4*>(&lds[slot + (wave + at) * 1024 + lane * 16]) = u32x4{0, 0, 0, 0};
      }
    }
  };
  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int m0 = wave / 2 * TM, w0 = wave % 2 * TN;
  const uint32_t swz = ((lane >> 4) ^ (lane & 7)) * 16;
  const uint32_t xat = (m0 + (lane & 15)) * 128 + swz, wat = (BM + w0 + (lane & 15)) * 128 + swz;
  for (int s = 0; s < D - 1 && s < stages; ++s) copy(s, s * STAGE);
  int slot = 0, to = (D - 1) * STAGE;
  for (int s = 0; s < stages; ++s) {
    // stage s is there; as many behind it as there are may still be on their way
    wait_stages<D - 2, LX + LW>(stages - 1 - s);
    lds_barrier();
    if (s + D - 1 < stages) copy(s + D - 1, to);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Vec xf[FM], wf[FN];
#pragma unroll
      for (int j = 0; j < FM; ++j) xf[j] = *reinterpret_cast<const Vec*>(&lds[slot + (xat ^ (64 * h)) + j * 2048]);
#pragma unroll
      for (int i = 0; i < FN; ++i) wf[i] = *reinterpret_cast<const Vec*>(&lds[slot + (wat ^ (64 * h)) + i * 2048]);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = dn_mfma(wf[i], xf[j], acc[i][j]);
    }
    to = slot;
    slot = slot + STAGE == D * STAGE ? 0 : slot + STAGE;
  }
  __syncthreads();
  dn_write<FM, FN>(p, w, m0, w0, acc, &lds[wave * kScratch<FN>]);
}

// The same product for rows at any alignment: stages pass through registers, four of
// them on their way there, into two in LDS.  Its loads are of 16 bytes at any element
// (dense_few_kernel's dwords were not tried here): they cost a third (K=2747 for 2752: 38
// and 28 us at M=1274 N=1520), the registers the rest (RING 64: 20); tiles of 128 are no
// faster (58).
template <int DT>
__global__ __launch_bounds__(256) void dense_ragged_kernel(const DenseP p) {
  using Vec = typename DnVec<DT>::type;
  constexpr int B = 64, AHEAD = 4, WAVES = 4, TM = B / 2, FM = TM / 16, FN = FM, LOADS = B / 8 / WAVES, UNIT = B * 128;
  __shared__ __align__(16) char lds[2 * 2 * UNIT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  const int m0 = wave / 2 * TM, w0 = wave % 2 * TM;
  const uint32_t swz = ((lane >> 4) ^ (lane & 7)) * 16;
  const uint32_t xat = (m0 + (lane & 15)) * 128 + swz, wat = UNIT + (w0 + (lane & 15)) * 128 + swz;
  struct Stage {
    u32x4 x[LOADS], w[LOADS];
  };
  auto load = [&](Stage& v, int s) {
    const int k = kfrom + s * DN_BK + 8 * piece;
    if (kfrom + (s + 1) * DN_BK <= kto) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        __builtin_memcpy(&v.w[i], wr[i] + k, 16);
        __builtin_memcpy(&v.x[i], x[i] + k, 16);
      }
    } else if (s < stages) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        v.w[i] = dn_load8<false>(wr[i], k, kto);
        v.x[i] = dn_load8<false>(x[i], k, kto);
      }
    }
  };
  auto turn = [&](Stage& v, int s) {  // v: stage s, then stage s + AHEAD
    char* buffer = lds + (s & 1) * 2 * UNIT;
    char* to = buffer + wave * 1024 + lane * 16;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      *reinterpret_cast<u32x4*>(to + i * WAVES * 1024) = v.x[i];
      *reinterpret_cast<u32x4*>(to + UNIT + i * WAVES * 1024) = v.w[i];
    }
    lds_barrier();  // (all waves have multiplied stage s - 1, so stage s + 1 may take its buffer)
    load(v, s + AHEAD);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Vec xf[FM], wf[FN];
#pragma unroll
      for (int j = 0; j < FM; ++j) xf[j] = *reinterpret_cast<const Vec*>(buffer + (xat ^ (64 * h)) + j * 2048);
#pragma unroll
      for (int i = 0; i < FN; ++i) wf[i] = *reinterpret_cast<const Vec*>(buffer + (wat ^ (64 * h)) + i * 2048);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = dn_mfma(wf[i], xf[j], acc[i][j]);
    }
  };
  Stage v[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(v[i], i);
  for (int s = 0; s < stages; s += AHEAD)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s + i < stages) turn(v[i], s + i);
  __syncthreads();
  dn_write<FM, FN>(p, w, m0, w0, acc, &lds[wave * kScratch<FN>]);
}

// The splits' sums added in order, four of them on their way at once, and the
// epilogue: 4 to 5 us of latency for a small batch (M=93 N=1407), then L2's rate.
__global__ __launch_bounds__(256) void dense_join_kernel(const DenseP p) {
  const int quads = p.half / 4, total = (int)p.M * quads;
  const int64_t split = p.M * p.P / 4;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const int row = i / quads, c = i - row * quads;
    const f32x4* part = reinterpret_cast<const f32x4*>(p.part) + (int64_t)row * (p.P / 4) + c;
    f32x4 g = {0.f, 0.f, 0.f, 0.f}, u = g;
    for (int s = 0; s < p.splits; s += 4, part += 4 * split) {
      f32x4 a[4], b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (s + k < p.splits) {
          a[k] = part[k * split];
          if (p.gated) b[k] = part[k * split + quads];
        }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (s + k < p.splits) {
          g += a[k];
          if (p.gated) u += b[k];
        }
    }
    dn_finish(p, row, 0, 4 * c, g, u);
  }
}

// Rows of x and w with K to whole pieces of 8 and zeros behind it, at aligned
// addresses: what makes an unaligned product one for the kernels with LDS copies
// (M=6628 K=657 N=2x1735 105 us on unaligned rows, 45 on aligned ones, the copy 6).
struct PadP {
  const uint16_t* from[2];
  uint16_t* to[2];
  int64_t rows[2], ld[2];  // rows 0: used as they are
  int K, Kp;
};
__global__ __launch_bounds__(256) void dense_pad_kernel(const PadP p) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < p.rows[0] + p.rows[1]; r += (int64_t)gridDim.x * 4) {
    const int which = r >= p.rows[0];
    const int64_t row = which ? r - p.rows[0] : r;
    const uint16_t* from = p.from[which] + row * p.ld[which];
    uint16_t* to = p.to[which] + row * p.Kp;
    for (int k = 8 * lane; k < p.Kp; k += 512) *reinterpret_cast<u32x4*>(to + k) = dn_load8<false>(from, k, p.K);
  }
}

// ------------------------------------------------------------- dispatch --
enum Kind { FEW, MID, RING, TILE, RAGGED };  // (numbered as ccq_dense_linear_kernel returns them)

struct Plan {
  Kind kind;
  int bm, bn;       // of the tile; FEW: 16 rows, 16 NF columns
  int splits, kchunk;
  bool pad;         // x and w are copied to aligned rows first
};

// What a stage of 64 columns takes in us, with up to one and two workgroups on a
// CU (0: there is room for one), and what a tile takes besides.  From K = 4096 and
// 2048 over M = 32 .. 2048, N = 2048 .. 14336 (K=N=4096: M=256 RING 64 22.4 us, 128 29.5,
// TILE 128 33.5; M=1024 52, 34, 36, RING 256 x 128 49; K=4096 N=14336: M=512 RING 256 x
// 128 63, TILE 128 74.6, 256 x 192 74, 256 81; M=1024 TILE 128 138, 256 96.5; M=172 K=11376
// N=9808: RING 64 131 us, 128 in three splits 101, 256 x 128 in three 84).  RAGGED from K of
// odd sizes, against copies and aligned tiles (M=1274 K=2747 N=1520 38 us, copies and RING 64 31;
// M=346 K=5468 N=4379 59, copies and RING 128 48; M=293 K=2355 N=1447 17.9 and 20.9; M=54 K=6003
// N=1305 13.5 and 21): over 78 products its choice takes 1.3 % more than the best of them.
struct Shape {
  Kind kind;
  int bm, bn;
  float one, two, tile;
};
constexpr Shape kShapes[] = {
    {MID, 32, 64, 0.25f, 0.40f, 2.f},    {RING, 64, 64, 0.35f, 0.45f, 2.5f},   {RING, 128, 128, 0.46f, 0.f, 4.f},
    {RING, 256, 128, 0.90f, 0.f, 5.f},   {TILE, 128, 128, 0.72f, 0.97f, 5.f},  {TILE, 256, 192, 1.05f, 0.f, 6.f},
    {TILE, 256, 224, 1.30f, 0.f, 6.f},   {TILE, 256, 256, 1.42f, 0.f, 7.f},    {RAGGED, 64, 64, 0.6f, 0.85f, 2.f},
};

float shape_time(const Shape& s, const DenseP& p, int64_t mtiles, int splits) {
  const int64_t stages = cdiv(cdiv(p.K, DN_BK), splits);
  const int64_t groups = mtiles * cdiv(p.W, s.bn) * splits, round = s.two > 0.f ? 512 : 256;
  const float full = s.two > 0.f ? s.two : s.one;
  const int64_t rest = groups % round;
  float t = (float)(groups / round) * (stages * full + s.tile);
  if (rest > 0) t += stages * (rest <= 256 ? s.one : full) + s.tile;
  // the partial sums' way out and back, and a launch
  if (splits > 1) t += 4.f + (float)splits * p.M * p.W * 8 / 4e6f;
  return t;
}

// The same for rows grouped by expert, whose workgroups end one by one: each expert
// leaves 0.6 of a tile more than its rows fill, and the last round counts half a round
// more.  The weights' way from memory costs every shape alike.  Over 150 products (8 to
// 256 experts of 1/2 to 450 rows, K = 304 .. 14336) its choice takes 1.1 % more than the
// best one (8 experts, 4096 -> 2 x 14336: 1024 rows TILE 256 x 192 403 us,
// TILE 128 588; 8, 14336 -> 4096: 384 rows RING 128 173, RING 64 232; 128, 2048 -> 2 x 768: 48
// rows each TILE 128 155, RING 64 173; 16 rows MID 139, TILE 128 147; 8, 2048 -> 784: 576 rows
// RING 64 14.4, TILE 128 28).
constexpr Shape kGroupShapes[] = {
    {MID, 32, 64, 0.30f, 0.46f, 1.f},    {RING, 64, 64, 0.36f, 0.50f, 2.f},  {RING, 128, 128, 0.45f, 0.f, 4.5f},
    {TILE, 128, 128, 0.67f, 0.93f, 3.5f}, {TILE, 256, 192, 0.88f, 0.f, 6.f}, {TILE, 256, 256, 1.16f, 0.f, 8.f},
};
float group_time(const Shape& s, const DenseP& p) {
  const float experts = (float)std::min<int64_t>(p.M, p.E), stages = (float)cdiv(p.K, DN_BK);
  const float groups = std::max(experts, (float)p.M / s.bm + 0.6f * experts) * cdiv(p.W, s.bn);
  const float round = s.two > 0.f ? 512 : 256, whole = stages * (s.two > 0.f ? s.two : s.one) + s.tile;
  if (groups <= round) return groups <= 256 ? stages * s.one + s.tile : whole;
  return (groups / round + 0.5f) * whole;
}

// rows: of the batch, or of an expert on average; dma: x and w are aligned; can_pad: they can be made so
Plan make_plan(const DenseP& p, int64_t rows, bool dma, bool can_pad) {
  Plan q = {FEW, 16, 16, 1, p.K, false};
  const bool grouped = p.offsets != nullptr;
  const float pad_time = 3.f + (float)(p.M + (grouped ? (int64_t)p.E : 1) * p.W) * p.K * 4 / 4.5e6f;
  // (few tiles do not fill the card: 10 of K=2432, T=2 N=320, MID 12.4 us, FEW 6.1; 96 of K=2048, T=4 N=2x768, 11.3
  // and 8.7; 192, T=8, 11.9 and 12.5; 256 of K=768 7.6 and 8.1; 384, T=16, 20.9 and 22.8; 128 of K=4096 18.6 and 14.8, 512
  // 55.5 and 54.1)
  if (grouped && (rows > 16 || (dma && std::min<int64_t>(p.M, p.E) * cdiv(p.W, 64) >= 160))) {
    // unaligned rows run at some 300 TFLOP/s, aligned ones at 700
    q.pad = !dma && can_pad && 2.f * p.M * p.W * p.K * 1.9e-9f > pad_time;
    if (!dma && !q.pad) {
      q.kind = RAGGED, q.bm = q.bn = 64;
      return q;
    }
    float best = 0.f;
    for (const Shape& s : kGroupShapes) {
      if (s.kind == RING && s.bm == 128 && rows < 32) continue;  // (67 experts of 17 rows, K=4064 N=2x576: 154 us, MID 130)
      const float t = group_time(s, p);
      if (best == 0.f || t < best) best = t, q.kind = s.kind, q.bm = s.bm, q.bn = s.bn;
    }
    return q;
  }
  if (rows <= 16) {
    // as many columns a workgroup as leave one for every second CU, where there are that many (M=1: K=2048 N=5632 16
    // columns 8.0 us, 32 7.3, 64 11.0; K=4096 N=14336 32, 31, 25.6; K=N=4096 8.3, 11.5, 17.5); groups of rows bring as many
    // workgroups as experts.  K is not split, so narrow outputs with long K leave CUs idle (M=16 K=14336 N=1024 27 us,
    // M=17 on MID in 16 splits 12; K=7168 N=64 14 and 11)
    const int64_t sets = cdiv(p.W, 16) * (grouped ? std::min<int64_t>(p.M, p.E) : 1);
    q.bn = sets >= 640 ? 64 : sets >= 320 || p.gated ? 32 : 16;
    return q;
  }
  float best = 0.f;
  for (const Shape& s : kShapes) {
    const bool pad = s.kind != RAGGED && !dma;
    if ((pad && !can_pad) || (s.kind == RAGGED && dma)) continue;
    if (p.gated && s.bn == 224) continue;  // a wave's 112 rows are no whole pairs of gate and up
    const int64_t stages = cdiv(p.K, DN_BK);
    for (int splits = 1; splits <= 16; ++splits) {
      if (splits > 1 && (stages / splits < 4 || (s.kind == TILE && s.bm == 256))) break;
      const float t = shape_time(s, p, cdiv(p.M, s.bm), splits) + (pad ? pad_time : 0.f);
      if (best == 0.f || t < best) {
        best = t;
        q = {s.kind, s.bm, s.bn, 1, p.K, pad};
        if (splits > 1) {
          q.kchunk = (int)(cdiv(stages, splits) * DN_BK);
          q.splits = (int)cdiv(p.K, q.kchunk);
        }
      }
    }
  }
  return q;
}

// tiles of a product: of groups as many as any offsets can make
int64_t col_tiles(const DenseP& p, const Plan& q) { return cdiv(p.N, p.gated ? q.bn / 2 : q.bn); }
int64_t row_tiles(const DenseP& p, const Plan& q) {
  return p.offsets == nullptr ? cdiv(p.M, q.bm) : imin64(p.M, p.E + 1) + p.M / q.bm;
}
int64_t workgroups(const DenseP& p, const Plan& q) { return row_tiles(p, q) * col_tiles(p, q) * q.splits; }
constexpr int64_t DN_MAX_TILES = 1 << 22;  // (of 512 threads, so that a launch stays below 2^32 of them)

template <int DT, int NF, int U, int WAVES>
void launch_few(const DenseP& p, dim3 grid, hipStream_t st) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w);
  if (at & 2 || p.K & 1 || (p.M > 1 && p.ldx & 1))
    launch(dense_few_kernel<DT, 1, NF, U, WAVES, ODD>, grid, dim3(64 * WAVES), 0, st, p);
  else if (p.K % 8 != 0)
    launch(dense_few_kernel<DT, 1, NF, U, WAVES, EVEN>, grid, dim3(64 * WAVES), 0, st, p);
  else
    launch(dense_few_kernel<DT, 1, NF, U, WAVES, WHOLE>, grid, dim3(64 * WAVES), 0, st, p);
}

template <int DT>
int launch_dense(DenseP p, const Plan& q, hipStream_t st, const char* what) {
  p.ntiles = (int)col_tiles(p, q);
  p.mtiles = (int)row_tiles(p, q);
  p.splits = q.splits;
  p.kchunk = q.splits > 1 ? q.kchunk : p.K;
  const dim3 grid((uint32_t)workgroups(p, q));
  if (q.kind == FEW) {
    if (q.bn == 16) launch_few<DT, 1, 4, 8>(p, grid, st);
    else if (q.bn == 32) launch_few<DT, 2, 4, 8>(p, grid, st);
    else launch_few<DT, 4, 2, 4>(p, grid, st);
  } else if (q.kind == MID) {
    launch(dense_mid_kernel<DT, 32, 64, 4>, grid, dim3(256), 0, st, p);
  } else if (q.kind == RING) {
    if (q.bm == 64) launch(dense_ring_kernel<DT, 64, 64, 2, 2, 3>, grid, dim3(256), 0, st, p);
    else if (q.bm == 128) launch(dense_ring_kernel<DT, 128, 128, 2, 4, 2>, grid, dim3(512), 0, st, p);
    else launch(dense_ring_kernel<DT, 256, 128, 4, 2, 2>, grid, dim3(512), 0, st, p);
  } else if (q.kind == TILE) {
    if (q.bm == 128) launch(dense_tile_kernel<DT, 128, 128, 2, 2>, grid, dim3(256), 0, st, p);
    else if (q.bn == 192) launch(dense_tile_kernel<DT, 256, 192, 4, 2>, grid, dim3(512), 0, st, p);
    else if (q.bn == 224) launch(dense_tile_kernel<DT, 256, 224, 4, 2>, grid, dim3(512), 0, st, p);
    else launch(dense_tile_kernel<DT, 256, 256, 4, 2>, grid, dim3(512), 0, st, p);
  } else {
    launch(dense_ragged_kernel<DT>, grid, dim3(256), 0, st, p);
  }
  if (int rc = launch_status(what)) return rc;
  if (p.part != nullptr) {
    launch(dense_join_kernel, dim3((uint32_t)grid_for(p.M * p.half / 4, 256)), dim3(256), 0, st, p);
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
  p.half = (int)(cdiv(a.N, 4) * 4), p.P = a.gated ? 2 * p.half : p.half;
  p.E = grouped ? (int)a.num_experts : 1;  // (a batch's one "expert" is 0)
  p.gated = a.gated != 0, p.act = a.act, p.bias_dtype = a.bias_dtype, p.y_dtype = a.y_dtype;
  return p;
}

// LDS copies: 16-byte pieces at 16-byte addresses, offsets from a tile's first row in 32 bits
bool in_reach(int64_t K, int64_t ldx, const ccq_dense_args& a) {
  return 256 * ldx + K < 1ll << 31 && ((a.gated ? a.N : 0) + 256) * K < 1ll << 31;
}
bool x_aligned(const ccq_dense_args& a) { return a.K % 8 == 0 && (a.M <= 1 || a.ldx % 8 == 0) && aligned(a.x, 16); }
bool w_aligned(const ccq_dense_args& a) { return a.K % 8 == 0 && aligned(a.w, 16); }

Plan plan_of(const ccq_dense_args& a, const DenseP& p) {
  const int64_t Kp = cdiv(a.K, 8) * 8;
  const bool dma = x_aligned(a) && w_aligned(a) && in_reach(a.K, a.M > 1 ? a.ldx : a.K, a);
  return make_plan(p, p.offsets != nullptr ? cdiv(a.M, a.num_experts) : a.M, dma, in_reach(Kp, std::max(Kp, a.ldx), a));
}

// the splits' sums, then the aligned rows of x and of w
struct Scratch {
  size_t part, x, w;
};
Scratch scratch_of(const ccq_dense_args& a, const DenseP& p, const Plan& q) {
  const size_t Kp = (size_t)cdiv(a.K, 8) * 8, L = p.offsets != nullptr ? (size_t)p.E : 1;
  const auto whole = [](size_t n) { return (n + 255) / 256 * 256; };
  return {q.splits > 1 ? whole((size_t)q.splits * p.M * p.P * 4) : 0, q.pad && !x_aligned(a) ? whole(p.M * Kp * 2) : 0,
          q.pad && !w_aligned(a) ? whole(L * p.W * Kp * 2) : 0};
}

size_t workspace_of(const char* what, const ccq_dense_args* args, bool grouped) {
  if (args == nullptr || args->M < 1 || check_dense(what, *args, grouped)) return 0;
  const DenseP p = make_params(*args, grouped);
  const Plan q = plan_of(*args, p);
  if (workgroups(p, q) >= DN_MAX_TILES) return 0;
  const Scratch s = scratch_of(*args, p, q);
  return s.part + s.x + s.w;
}

int run_dense(const char* what, const ccq_dense_args* args, bool grouped) {
  CCQ_REQUIRE(args != nullptr, "%s: null arguments", what);
  const ccq_dense_args& a = *args;
  if (int rc = check_dense(what, a, grouped)) return rc;
  if (a.M == 0) return 0;
  DenseP p = make_params(a, grouped);
  const Plan q = plan_of(a, p);
  CCQ_REQUIRE(workgroups(p, q) < DN_MAX_TILES, "%s: M=%lld, N=%lld in %lld tiles, fewer than 2^22 tiles fit a launch", what,
              (long long)a.M, (long long)a.N, (long long)workgroups(p, q));
  const Scratch s = scratch_of(a, p, q);
  const size_t need = s.part + s.x + s.w;
  CCQ_REQUIRE(need == 0 || (a.workspace != nullptr && aligned(a.workspace, 16) && a.workspace_bytes >= need),
              "%s: workspace of %zu bytes needed", what, need);
  char* at = reinterpret_cast<char*>(a.workspace);
  const hipStream_t st = as_stream(a.stream);
  if (s.part) p.part = reinterpret_cast<float*>(at);
  if (q.pad) {
    PadP pad = {};
    pad.K = p.K, pad.Kp = (int)(cdiv(a.K, 8) * 8);
    if (s.x) {
      pad.from[0] = reinterpret_cast<const uint16_t*>(a.x), pad.to[0] = reinterpret_cast<uint16_t*>(at + s.part);
      pad.rows[0] = p.M, pad.ld[0] = a.ldx;
      p.x = pad.to[0], p.ldx = pad.Kp;
    }
    if (s.w) {
      pad.from[1] = reinterpret_cast<const uint16_t*>(a.w), pad.to[1] = reinterpret_cast<uint16_t*>(at + s.part + s.x);
      pad.rows[1] = (grouped ? (int64_t)p.E : 1) * p.W, pad.ld[1] = p.K;
      p.w = pad.to[1];
    }
    p.K = pad.Kp;
    launch(dense_pad_kernel, dim3((uint32_t)std::min<int64_t>(cdiv(pad.rows[0] + pad.rows[1], 4), 8192)), dim3(256), 0, st, pad);
    if (int rc = launch_status(what)) return rc;
  }
  return a.dtype == CCQ_BF16 ? launch_dense<CCQ_BF16>(p, q, st, what) : launch_dense<CCQ_F16>(p, q, st, what);
}

}  // namespace

}  // namespace ccq

using namespace ccq;

extern "C" size_t ccq_dense_linear_workspace_size(const ccq_dense_args* args) {
  return workspace_of("ccq_dense_linear", args, false);
}

extern "C" int ccq_dense_linear_kernel(const ccq_dense_args* args, int grouped, int* tile_rows, int* tile_cols, int* splits,
                                       int* copies) {
  const char* what = grouped ? "ccq_dense_linear_grouped" : "ccq_dense_linear";
  Plan q = {};
  int kernel = -1, copied = 0;
  if (args != nullptr && args->M >= 1 && check_dense(what, *args, grouped != 0) == 0) {
    const DenseP p = make_params(*args, grouped != 0);
    const Plan plan = plan_of(*args, p);
    if (workgroups(p, plan) < DN_MAX_TILES) {
      const Scratch s = scratch_of(*args, p, plan);
      q = plan, kernel = q.kind, copied = (s.x ? 1 : 0) | (s.w ? 2 : 0);
    }
  }
  if (tile_rows) *tile_rows = q.bm;
  if (tile_cols) *tile_cols = q.bn;
  if (splits) *splits = q.splits;
  if (copies) *copies = copied;
  return kernel;
}

extern "C" int ccq_dense_linear(const ccq_dense_args* args) { return run_dense("ccq_dense_linear", args, false); }

extern "C" size_t ccq_dense_linear_grouped_workspace_size(const ccq_dense_args* args) {
  return workspace_of("ccq_dense_linear_grouped", args, true);
}

extern "C" int ccq_dense_linear_grouped(const ccq_dense_args* args) {
  return run_dense("ccq_dense_linear_grouped", args, true);
}
