// Low-rank adapters of many requests beside one shared projection:
//   y[t] += scale[i] * B_i (A_i x[t]),  i = index[t],
// A [L, R, K], B [L, N, R] in 16 bits, products and sums in float32, y rounded
// once.  Rows whose index is outside [0, L) are not touched.
//
// The tokens are sorted by adapter into tiles of 16 (the expert schedule of
// ccq_moe_align), then two products run on the matrix cores:
//   shrink  p[t, r] = sum_k x[t, k] A[i, r, k], K split over workgroups and
//           waves, each split's sums in its own part of the workspace;
//   expand  y[t, n] += sum_r (scale * p[t, r]) B[i, n, r], the splits of p
//           added in their order.
#include "ccq_common.h"

#include <math.h>

#include <type_traits>

namespace ccq {

namespace {

constexpr int LR_TM = 16;       // tokens of a tile
constexpr int LR_MAX_R = 256;
constexpr int LR_MAX_S = 64;

struct LoraP {
  const void* x;
  void* y;
  const void* a;
  const void* b;
  const float* scale;
  const int32_t* rank;
  const int32_t* sorted_ids;
  const int32_t* tile_adapter;
  const int32_t* meta;
  float* p;                     // [S][T][Rp]
  int64_t ldx, ldy, T;
  int R, Rp, K, N, S, kchunk;   // kchunk: K per wave, a multiple of 32
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

// 8 consecutive 16-bit values at any alignment, those from n on as 0
__device__ __forceinline__ u32x4 lr_load16(const void* base, int64_t i, int n) {
  const uint16_t* h = reinterpret_cast<const uint16_t*>(base) + i;
  u32x4 v = {0, 0, 0, 0};
  if (n >= 8) {
    __builtin_memcpy(&v, h, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) v[e >> 1] |= (uint32_t)h[e] << (16 * (e & 1));
  }
  return v;
}

template <int DT>
__device__ __forceinline__ void lr_load_f32(const void* base, int64_t i, int n, float (&v)[8]) {
  if constexpr (DT == CCQ_F32) {
    const float* f = reinterpret_cast<const float*>(base) + i;
    if (n >= 8) {
      __builtin_memcpy(v, f, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? f[e] : 0.f;
    }
  } else {
    const u32x4 b = lr_load16(base, i, n);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t u = (b[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
      v[e] = DT == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
    }
  }
}

__device__ __forceinline__ int lr_rank(const LoraP& p, int adapter) {
  return p.rank != nullptr ? min(max(p.rank[adapter], 0), p.R) : p.R;
}

// ------------------------------------------------------------------ shrink --
// One workgroup: a tile's 16 tokens, RT * 16 ranks from 16 RT blockIdx.z, the
// K range of split blockIdx.y, a quarter of it per wave.  16x16x32 MFMA: A
// operand lane = token, B operand lane = rank, both with k = 8 (lane >> 4) + e
// (16-bit x and A of one type); else the same values in float32 on 16x16x4,
// element e of every lane in one instruction.
template <int XT, int WT, int RT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraP p) {
  constexpr bool NATIVE = XT == WT;
  const int tile = blockIdx.x;
  if (tile >= p.meta[0]) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int adapter = p.tile_adapter[tile];
  const int rank = lr_rank(p, adapter), r0 = blockIdx.z * RT * 16;
  if (r0 >= rank) return;
  const int own = p.sorted_ids[tile * LR_TM + c16];
  const int tok = own >= 0 ? own : p.sorted_ids[tile * LR_TM];  // padding: the first row again, not stored
  const int64_t xrow = (int64_t)tok * p.ldx;
  int64_t arow[RT];
  bool live[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + t * 16 + c16;
    live[t] = r < rank;
    arow[t] = ((int64_t)adapter * p.R + r) * p.K;
  }
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int k0 = (blockIdx.y * 4 + wave) * p.kchunk, k1 = min(k0 + p.kchunk, p.K);
  for (int k = k0; k < k1; k += 32) {
    const int kk = k + 8 * g, n = p.K - kk;
    if constexpr (NATIVE) {
      using V = typename Half<WT>::vec;
      const V xv = __builtin_bit_cast(V, lr_load16(p.x, xrow + kk, n));
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const V av = __builtin_bit_cast(V, lr_load16(p.a, arow[t] + kk, live[t] ? n : 0));
        acc[t] = lr_mfma(xv, av, acc[t]);
      }
    } else {
      float xv[8], av[8];
      lr_load_f32<XT>(p.x, xrow + kk, n, xv);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        lr_load_f32<WT>(p.a, arow[t] + kk, live[t] ? n : 0, av);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[e], av[e], acc[t], 0, 0, 0);
      }
    }
  }
  __shared__ f32x4 red[4][RT][64];
#pragma unroll
  for (int t = 0; t < RT; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < RT; t += 4) {
    if (r0 + t * 16 >= rank) break;
    const f32x4 s = ((red[0][t][lane] + red[1][t][lane]) + red[2][t][lane]) + red[3][t][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // D: column (rank) lane & 15, row (token) 4 (lane >> 4) + i
      const int id = p.sorted_ids[tile * LR_TM + 4 * g + i];
      if (id >= 0) p.p[((int64_t)blockIdx.y * p.T + id) * p.Rp + r0 + t * 16 + c16] = s[i];
    }
  }
}

// ------------------------------------------------------------------ expand --
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

template <int YT>
__device__ __forceinline__ float lr_load1(const void* y, int64_t i) {
  if constexpr (YT == CCQ_F32) return reinterpret_cast<const float*>(y)[i];
  const uint32_t u = reinterpret_cast<const uint16_t*>(y)[i];
  return YT == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
}
template <int YT>
__device__ __forceinline__ void lr_store1(void* y, int64_t i, float v) {
  if constexpr (YT == CCQ_F32)
    reinterpret_cast<float*>(y)[i] = v;
  else
    reinterpret_cast<uint16_t*>(y)[i] = (uint16_t)(YT == CCQ_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
}

// One wave: a tile's 16 tokens x 64 columns.  The A operand of MFMA q is the
// 16 rows n0 + 16 (m >> 2) + 4 q + (m & 3) of B, m = lane & 15, the B operand
// p (lane & 15 = token), so lane (g, token) ends with the 16 consecutive
// columns n0 + 16 g + (4 q + i) of its token.
template <int WT, int YT>
__global__ __launch_bounds__(256) void lora_expand_kernel(const LoraP p) {
  using V = typename Half<WT>::vec;
  constexpr int PARTS = WT == CCQ_BF16 && YT == CCQ_F32 ? 3 : 2;
  const int tile = blockIdx.y;
  if (tile >= p.meta[0]) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int n0 = (blockIdx.x * 4 + wave) * 64;
  if (n0 >= p.N) return;
  const int adapter = p.tile_adapter[tile];
  const int rank = lr_rank(p, adapter);
  if (rank == 0) return;
  const float scale = p.scale != nullptr ? p.scale[adapter] : 1.f;
  const int own = p.sorted_ids[tile * LR_TM + c16];
  const int64_t tok = own >= 0 ? own : p.sorted_ids[tile * LR_TM];
  f32x4 acc[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
  float up = 1.f, down = 1.f;  // f16: the row's power of two, and its inverse
  auto load_p = [&](int r, float(&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (r >= ((rank + 15) & ~15)) return;
    for (int s = 0; s < p.S; ++s) {
      float u[8];
      __builtin_memcpy(u, p.p + ((int64_t)s * p.T + tok) * p.Rp + r, 32);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += u[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= scale;
  };
  if constexpr (WT == CCQ_F16) {
    float m = 0.f;
    for (int c = 0; c < rank; c += 32) {
      float v[8];
      load_p(c + 8 * g, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = isfinite(v[e]) ? fmaxf(m, fabsf(v[e])) : m;
    }
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if (m > 0.f) {
      const int e = min(max(14 - ilogbf(m), -100), 100);
      up = ldexpf(1.f, e);
      down = ldexpf(1.f, -e);
    }
  }
  for (int c = 0; c < rank; c += 32) {
    const int r = c + 8 * g;
    float v[8];
    V pv[PARTS];
    load_p(r, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= up;
    lr_split<WT, PARTS>(v, pv);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + 16 * (c16 >> 2) + 4 * q + (c16 & 3);
      const V bv = __builtin_bit_cast(
          V, lr_load16(p.b, ((int64_t)adapter * p.N + n) * p.R + r, n < p.N ? rank - r : 0));
#pragma unroll
      for (int i = 0; i < PARTS; ++i) acc[q] = lr_mfma(bv, pv[i], acc[q]);
    }
  }
  if (own < 0) return;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 16 * g + 4 * q + i;
      if (n < p.N) {
        const int64_t at = tok * p.ldy + n;
        lr_store1<YT>(p.y, at, lr_load1<YT>(p.y, at) + acc[q][i] * down);
      }
    }
}

size_t a256l(size_t b) { return (b + 255) & ~(size_t)255; }

struct LoraLayout {
  int64_t max_tiles, S, kchunk, Rp;
  size_t off_sorted, off_tile, off_meta, off_counts, off_align, off_p, total;
};

LoraLayout lora_layout(int64_t T, const ccq_lora_adapters* ad) {
  LoraLayout L = {};
  L.max_tiles = ccq_moe_align_max_tiles(T, ad->num_adapters, LR_TM);
  L.Rp = cdiv(ad->rank_max, 16) * 16;
  // K over enough workgroups for two on each of the 256 CUs, at least 128 per wave
  const int64_t most = cdiv(ad->in_features, 4 * 128);
  int64_t S = cdiv(512, L.max_tiles);
  S = S < most ? S : most;
  S = S < LR_MAX_S ? S : LR_MAX_S;
  L.kchunk = cdiv(cdiv(ad->in_features, 4 * S), 32) * 32;
  L.S = cdiv(ad->in_features, 4 * L.kchunk);
  size_t o = 0;
  L.off_sorted = o;
  o += a256l((size_t)L.max_tiles * LR_TM * 4);
  L.off_tile = o;
  o += a256l((size_t)L.max_tiles * 4);
  L.off_meta = o;
  o += 256;
  L.off_counts = o;
  o += a256l((size_t)ad->num_adapters * 4);
  L.off_align = o;
  o += a256l(align_scratch_bytes(T, ad->num_adapters));
  L.off_p = o;
  o += a256l((size_t)L.S * T * L.Rp * 4);
  L.total = o;
  return L;
}

int check_adapters(const ccq_lora_adapters* ad, const char* name) {
  CCQ_REQUIRE(ad != nullptr, "%s: null adapter descriptor", name);
  CCQ_REQUIRE(ad->dtype == CCQ_F16 || ad->dtype == CCQ_BF16, "%s: adapters must be f16 or bf16", name);
  CCQ_REQUIRE(ad->num_adapters >= 1 && ad->num_adapters <= 1024, "%s: num_adapters=%lld outside [1, 1024]", name,
              (long long)ad->num_adapters);
  CCQ_REQUIRE(ad->rank_max >= 1 && ad->rank_max <= LR_MAX_R, "%s: rank_max=%lld outside [1, %d]", name,
              (long long)ad->rank_max, LR_MAX_R);
  CCQ_REQUIRE(ad->in_features >= 1 && ad->in_features <= (1 << 20) && ad->out_features >= 1 &&
                  ad->out_features <= (1 << 20),
              "%s: in_features=%lld and out_features=%lld must be in [1, 2^20]", name, (long long)ad->in_features,
              (long long)ad->out_features);
  return 0;
}

template <int XT, int WT>
void shrink_launch(const LoraP& p, int64_t tiles, hipStream_t st) {
  const int rt = (int)cdiv(p.R, 16);
  const dim3 block(256);
  const unsigned x = (unsigned)tiles, y = (unsigned)p.S;
  if (rt <= 1)
    launch((lora_shrink_kernel<XT, WT, 1>), dim3(x, y, 1), block, 0, st, p);
  else if (rt <= 2)
    launch((lora_shrink_kernel<XT, WT, 2>), dim3(x, y, 1), block, 0, st, p);
  else if (rt <= 4)
    launch((lora_shrink_kernel<XT, WT, 4>), dim3(x, y, 1), block, 0, st, p);
  else
    launch((lora_shrink_kernel<XT, WT, 8>), dim3(x, y, (unsigned)cdiv(rt, 8)), block, 0, st, p);
}

template <int WT>
void expand_launch(const LoraP& p, int y_dtype, int64_t tiles, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(p.N, 256), (unsigned)tiles), block(256);
  if (y_dtype == CCQ_F32)
    launch((lora_expand_kernel<WT, CCQ_F32>), grid, block, 0, st, p);
  else if (y_dtype == CCQ_F16)
    launch((lora_expand_kernel<WT, CCQ_F16>), grid, block, 0, st, p);
  else
    launch((lora_expand_kernel<WT, CCQ_BF16>), grid, block, 0, st, p);
}

bool lora_float_code(int dt) { return dt == CCQ_F32 || dt == CCQ_F16 || dt == CCQ_BF16; }

}  // namespace

}  // namespace ccq

using namespace ccq;

extern "C" size_t ccq_lora_workspace_size(int64_t T, const ccq_lora_adapters* ad) {
  if (T <= 0 || T > 65536 || check_adapters(ad, "ccq_lora_workspace_size")) return 0;
  return lora_layout(T, ad).total;
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
  const LoraLayout L = lora_layout(T, ad);
  CCQ_REQUIRE(workspace && workspace_bytes >= L.total && aligned(workspace, 256),
              "ccq_lora_add: workspace of %zu bytes (256-byte aligned) needed, %zu given", L.total, workspace_bytes);
  hipStream_t st = as_stream(stream);
  char* ws = (char*)workspace;
  int rc = launch_align(index, T, ad->num_adapters, LR_TM, (int32_t*)(ws + L.off_sorted), (int32_t*)(ws + L.off_tile),
                        (int32_t*)(ws + L.off_meta), (int32_t*)(ws + L.off_counts), st, ws + L.off_align,
                        align_scratch_bytes(T, ad->num_adapters));
  if (rc) return rc;
  LoraP p = {};
  p.x = x;
  p.y = y;
  p.a = ad->a;
  p.b = ad->b;
  p.scale = ad->scale;
  p.rank = ad->rank;
  p.sorted_ids = (const int32_t*)(ws + L.off_sorted);
  p.tile_adapter = (const int32_t*)(ws + L.off_tile);
  p.meta = (const int32_t*)(ws + L.off_meta);
  p.p = (float*)(ws + L.off_p);
  p.ldx = ldx;
  p.ldy = ldy;
  p.T = T;
  p.R = (int)ad->rank_max;
  p.Rp = (int)L.Rp;
  p.K = (int)ad->in_features;
  p.N = (int)ad->out_features;
  p.S = (int)L.S;
  p.kchunk = (int)L.kchunk;
  if (ad->dtype == CCQ_BF16) {
    if (x_dtype == CCQ_BF16)
      shrink_launch<CCQ_BF16, CCQ_BF16>(p, L.max_tiles, st);
    else if (x_dtype == CCQ_F16)
      shrink_launch<CCQ_F16, CCQ_BF16>(p, L.max_tiles, st);
    else
      shrink_launch<CCQ_F32, CCQ_BF16>(p, L.max_tiles, st);
    if ((rc = launch_status("ccq_lora_add (shrink)"))) return rc;
    expand_launch<CCQ_BF16>(p, y_dtype, L.max_tiles, st);
  } else {
    if (x_dtype == CCQ_BF16)
      shrink_launch<CCQ_BF16, CCQ_F16>(p, L.max_tiles, st);
    else if (x_dtype == CCQ_F16)
      shrink_launch<CCQ_F16, CCQ_F16>(p, L.max_tiles, st);
    else
      shrink_launch<CCQ_F32, CCQ_F16>(p, L.max_tiles, st);
    if ((rc = launch_status("ccq_lora_add (shrink)"))) return rc;
    expand_launch<CCQ_F16>(p, y_dtype, L.max_tiles, st);
  }
  return launch_status("ccq_lora_add (expand)");
}
