// Tokens sorted by expert and back, and the gradients of both.
//
// Assignment a = t k + s gives token t to expert ids[a]; key(a) is that expert,
// or E where ids[a] is outside [0, E).  The order is by (key, a):
//   position[a] = #{a' : (key(a'), a') < (key(a), a)}, as ~row where key(a) = E,
//   offsets[e]  = #{a' : key(a') < e},  e = 0 .. E,
//   permute     rows[position[t, s]] = x[t], zero from row offsets[E] on,
//   unpermute   y[t] = sum_s weights[t, s] rows[position[t, s]]  (kept s, in order, float32),
//   its gradient  d_rows[position[t, s]] = weights[t, s] dy[t],
//                 d_weights[t, s] = sum_h rows[position[t, s], h] dy[t, h]  (float32).
// The gradient of permute is unpermute without weights.
//
// A permutation of no arithmetic to speak of: bytes bound it.  Everything goes by
// tokens, so that a token's row is read once and its k rows are written (or read)
// from there, 16 bytes a lane.
#include "ccq_common.h"

#include <algorithm>

namespace ccq {

namespace {

constexpr int PM_THREADS = 256, PM_WAVES = 4;
constexpr int PM_MAX_E = 1024, PM_KEY_BITS = 11;
constexpr int PM_MAX_K = 64;
constexpr int64_t PM_MAX_N = 1 << 20;
constexpr int PM_OWN = 256;            // most assignments of a workgroup
constexpr int PM_CHUNK = 512;          // assignments of a row of counts
constexpr int PM_SCAN_WAVES = 16;
// Most assignments that every workgroup ranks its own among by itself, in one
// launch; more of them go by counts of chunks, in three (H=2048, k=8: T=128 5.7 us, by
// chunks 9.6; T=256 8.1 and 10.7; T=512 13.8 and 12.1).
constexpr int PM_SELF = 2048, PM_SHIFT = 20;

struct PermP {
  const void* x;
  const int64_t* ids;
  void* rows;
  int32_t* position;
  int32_t* offsets;
  int32_t* table;                      // [chunks][E + 1] counts, then those of all chunks before
  int32_t* total;                      // [E + 1]
  int64_t ldx;                         // bytes
  int64_t T;
  int n, k, E, H, esize;
  int tokens;                          // of a workgroup
  int chunks;
};

__device__ __forceinline__ uint32_t pm_key(const PermP& p, int a) {
  const int64_t id = p.ids[a];
  return id >= 0 && id < p.E ? (uint32_t)id : (uint32_t)p.E;
}

struct PermS {
  int total[PM_MAX_E + 1], start[PM_MAX_E + 1];
  int sum[PM_WAVES];
  uint32_t own[PM_OWN];
  int rank[PM_OWN];
};
// s.total (counts by key) -> s.start (rows before a key), by all threads
__device__ __forceinline__ void pm_starts(const PermP& p, PermS& s) {
  constexpr int PER = (PM_MAX_E + 1 + PM_THREADS - 1) / PM_THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int v[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = tid * PER + i;
    v[i] = e <= p.E ? s.total[e] : 0;
    sum += v[i];
  }
  int at = wave_scan(sum);
  if (lane == 63) s.sum[wave] = at;
  __syncthreads();
  at -= sum;
#pragma unroll
  for (int w = 0; w < PM_WAVES - 1; ++w) at += w < wave ? s.sum[w] : 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = tid * PER + i;
    if (e <= p.E) s.start[e] = at;
    at += v[i];
  }
  __syncthreads();
}

// One 16-byte piece of a row, at any alignment of the elements (a row's last
// piece ends with the row and may repeat some of the one before).
__device__ __forceinline__ u32x4 pm_load(const char* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ void pm_store(char* p, u32x4 v) { __builtin_memcpy(p, &v, 16); }

// Tokens t0 .. t0 + tokens - 1 to the rows rank[j] (~row: zeros) of their assignments,
// four pieces of a thread on their way.
__device__ __forceinline__ void pm_copy(const PermP& p, const int* rank, int64_t t0, int tokens) {
  const int tid = threadIdx.x;
  const int64_t width = (int64_t)p.H * p.esize;
  const char* x = reinterpret_cast<const char*>(p.x) + t0 * p.ldx;
  char* rows = reinterpret_cast<char*>(p.rows);
  if (width < 16) {
    for (int j = tid; j < tokens * p.k; j += PM_THREADS) {
      const int at = rank[j];
      char* row = rows + (int64_t)(at < 0 ? ~at : at) * width;
      for (int b = 0; b < width; b += 2)
        *reinterpret_cast<uint16_t*>(row + b) =
            at < 0 ? (uint16_t)0 : *reinterpret_cast<const uint16_t*>(x + j / p.k * p.ldx + b);
    }
    return;
  }
  const uint32_t pieces = (uint32_t)((width + 15) / 16), all = tokens * pieces;
  for (uint32_t base = tid; base < all; base += 4 * PM_THREADS) {
    u32x4 v[4];
    int64_t at[4];
    int first[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = base + i * PM_THREADS;
      if (u >= all) continue;
      const uint32_t t = u / pieces;
      at[i] = imin64(16ll * (u - t * pieces), width - 16);
      first[i] = t * p.k;
      v[i] = pm_load(x + t * p.ldx + at[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (base + i * PM_THREADS >= all) continue;
      for (int s = 0; s < p.k; ++s) {
        const int row = rank[first[i] + s];
        pm_store(rows + (int64_t)(row < 0 ? ~row : row) * width + at[i], row < 0 ? u32x4{0, 0, 0, 0} : v[i]);
      }
    }
  }
}

// Up to PM_SELF assignments: workgroup b sorts and copies `tokens` tokens; the last
// one writes the offsets.  A workgroup needs the rank of its own few assignments
// only, which it finds by comparing them with all others: a ballot a comparison, no
// sort, and for a decode batch no second launch.
__global__ __launch_bounds__(PM_THREADS) void permute_kernel(const PermP p) {
  __shared__ PermS s;
  const int tid = threadIdx.x, lane = tid & 63;
  if (blockIdx.x == gridDim.x - 1) {
    for (int e = tid; e <= p.E; e += PM_THREADS) s.total[e] = 0;
    __syncthreads();
    for (int a = tid; a < p.n; a += PM_THREADS) atomicAdd(&s.total[pm_key(p, a)], 1);
    __syncthreads();
    pm_starts(p, s);
    for (int e = tid; e <= p.E; e += PM_THREADS) p.offsets[e] = s.start[e];
    return;
  }
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int tokens = (int)imin64(p.tokens, p.T - t0);
  const int a0 = (int)t0 * p.k, own = tokens * p.k;
  for (int j = tid; j < own; j += PM_THREADS) {
    s.own[j] = pm_key(p, a0 + j) << PM_SHIFT | (uint32_t)(a0 + j);
    s.rank[j] = 0;
  }
  __syncthreads();
  for (int base = 0; base < p.n; base += 4 * PM_THREADS) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = base + i * PM_THREADS + tid;
      c[i] = a < p.n ? pm_key(p, a) << PM_SHIFT | (uint32_t)a : ~0u;
    }
    for (int j = 0; j < own; ++j) {
      const uint32_t mine = __builtin_amdgcn_readfirstlane(s.own[j]);
      int count = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) count += __builtin_popcountll(__ballot(c[i] < mine));
      if (lane == 0 && count) atomicAdd(&s.rank[j], count);
    }
  }
  __syncthreads();
  for (int j = tid; j < own; j += PM_THREADS) {
    if ((int)(s.own[j] >> PM_SHIFT) == p.E) s.rank[j] = ~s.rank[j];
    p.position[a0 + j] = s.rank[j];
  }
  __syncthreads();
  pm_copy(p, s.rank, t0, tokens);
}

// More of them.  First, a chunk's counts of each expert, and into position each
// assignment's rank among the chunk's of its expert.  A wave takes 64 assignments at
// a time: eleven ballots on the bits of their keys leave each lane the lanes of its
// own key, those below it count, and the first of them adds them all to the wave's
// counts.
__global__ __launch_bounds__(PM_THREADS) void permute_rank_kernel(const PermP p) {
  constexpr int TURNS = PM_CHUNK / PM_THREADS;
  __shared__ int count[PM_WAVES][PM_MAX_E + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int e = tid; e <= p.E; e += PM_THREADS)
#pragma unroll
    for (int w = 0; w < PM_WAVES; ++w) count[w][e] = 0;
  const int a0 = blockIdx.x * PM_CHUNK + wave * (PM_CHUNK / PM_WAVES) + lane;
  uint32_t key[TURNS];
  int rank[TURNS];
#pragma unroll
  for (int i = 0; i < TURNS; ++i) key[i] = a0 + 64 * i < p.n ? pm_key(p, a0 + 64 * i) : PM_MAX_E + 1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    uint64_t same = ~0ull;
#pragma unroll
    for (int b = 0; b < PM_KEY_BITS; ++b) {
      const uint64_t set = __ballot(key[i] >> b & 1);
      same &= key[i] >> b & 1 ? set : ~set;
    }
    const int below = __builtin_popcountll(same & ((1ull << lane) - 1));
    if (key[i] <= PM_MAX_E) rank[i] = count[wave][key[i]] + below;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (key[i] <= PM_MAX_E && below == 0) count[wave][key[i]] = rank[i] + __builtin_popcountll(same);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    if (key[i] > PM_MAX_E) continue;
#pragma unroll
    for (int w = 0; w < PM_WAVES - 1; ++w) rank[i] += w < wave ? count[w][key[i]] : 0;
    p.position[a0 + 64 * i] = rank[i];
  }
  for (int e = tid; e <= p.E; e += PM_THREADS) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < PM_WAVES; ++w) sum += count[w][e];
    p.table[(int64_t)blockIdx.x * (p.E + 1) + e] = sum;
  }
}

// The counts of 64 experts a workgroup to those of all chunks before, and to their
// totals; its waves share the chunks.
__global__ __launch_bounds__(64 * PM_SCAN_WAVES) void permute_scan_kernel(const PermP p) {
  __shared__ int sums[PM_SCAN_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
  const int per = (p.chunks + PM_SCAN_WAVES - 1) / PM_SCAN_WAVES, from = wave * per, to = min(from + per, p.chunks);
  int32_t* column = p.table + e;
  const int64_t line = p.E + 1;
  int sum = 0;
  if (e <= p.E)
#pragma unroll 8
    for (int c = from; c < to; ++c) sum += column[c * line];
  sums[wave][lane] = sum;
  __syncthreads();
  if (e > p.E) return;
  int at = 0;
#pragma unroll
  for (int w = 0; w < PM_SCAN_WAVES; ++w) at += w < wave ? sums[w][lane] : 0;
  if (wave == PM_SCAN_WAVES - 1) p.total[e] = at + sum;
  for (int c0 = from; c0 < to; c0 += 8) {
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < to ? column[(c0 + i) * line] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c0 + i < to) column[(c0 + i) * line] = at;
      at += v[i];
    }
  }
}

// Then the rows; the last workgroup writes the offsets.  T=4096 k=8: H=2048 33 us for
// all three kernels, 4.6 TB/s; H=7168 105 us, 5.0 (the counts of all chunks read by every
// workgroup, and its assignments ranked there: 48 and 138); T=65536 H=2048 498 us, 4.9.
__global__ __launch_bounds__(PM_THREADS) void permute_copy_kernel(const PermP p) {
  __shared__ PermS s;
  const int tid = threadIdx.x;
  for (int e = tid; e <= p.E; e += PM_THREADS) s.total[e] = p.total[e];
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int tokens = blockIdx.x == gridDim.x - 1 ? 0 : (int)imin64(p.tokens, p.T - t0);
  const int a = (int)t0 * p.k + tid;
  uint32_t key = 0;
  int row = 0;
  static_assert(PM_OWN <= PM_THREADS, "an assignment a thread");
  if (tid < tokens * p.k) {
    key = pm_key(p, a);
    row = p.position[a] + p.table[(int64_t)(a / PM_CHUNK) * (p.E + 1) + key];
  }
  __syncthreads();
  pm_starts(p, s);
  if (blockIdx.x == gridDim.x - 1) {
    for (int e = tid; e <= p.E; e += PM_THREADS) p.offsets[e] = s.start[e];
    return;
  }
  if (tid < tokens * p.k) {
    row += s.start[key];
    s.rank[tid] = p.position[a] = (int)key == p.E ? ~row : row;
  }
  __syncthreads();
  pm_copy(p, s.rank, t0, tokens);
}

// --------------------------------------------------------------- and back --
struct UnpermP {
  const void* rows;
  const int32_t* position;
  const float* weights;  // or null
  const void* dy;        // gradients only
  void* out;             // y, or d_rows
  float* d_weights;
  int64_t ldr, ldy, R, T;  // strides in elements
  int k, H;
  int y_dtype;
  int pieces;            // threads on a token
  int64_t turn;          // tokens of a row of the grid
};

template <int DT>
constexpr int kPiece = DT == CCQ_F32 ? 4 : 8;  // elements of 16 bytes

template <int DT>
__device__ __forceinline__ void pm_floats(u32x4 b, float (&v)[kPiece<DT>]) {
#pragma unroll
  for (int e = 0; e < kPiece<DT>; ++e) {
    if constexpr (DT == CCQ_F32) {
      v[e] = __uint_as_float(b[e]);
    } else {
      const uint32_t u = (b[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
      v[e] = DT == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
    }
  }
}
__device__ __forceinline__ uint32_t pm_pair(int dt, float a, float b) {
  return dt == CCQ_BF16 ? bf16x2_bits(a, b) : f32_to_f16_bits(a) | f32_to_f16_bits(b) << 16;
}
template <int N>
__device__ __forceinline__ void pm_store_floats(int dt, void* y, int64_t i, const float (&v)[N]) {
  if (dt == CCQ_F32) {
    __builtin_memcpy(reinterpret_cast<float*>(y) + i, v, 4 * N);
  } else {
    uint32_t b[N / 2];
#pragma unroll
    for (int e = 0; e < N / 2; ++e) b[e] = pm_pair(dt, v[2 * e], v[2 * e + 1]);
    __builtin_memcpy(reinterpret_cast<uint16_t*>(y) + i, b, 2 * N);
  }
}
template <int DT>
__device__ __forceinline__ float pm_one(const void* p, int64_t i) {
  if constexpr (DT == CCQ_F32) return reinterpret_cast<const float*>(p)[i];
  const uint32_t u = reinterpret_cast<const uint16_t*>(p)[i];
  return DT == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
}
__device__ __forceinline__ void pm_store_one(int dt, void* y, int64_t i, float v) {
  if (dt == CCQ_F32)
    reinterpret_cast<float*>(y)[i] = v;
  else
    reinterpret_cast<uint16_t*>(y)[i] = (uint16_t)(dt == CCQ_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
}

// A thread adds one piece of a token's rows, eight of them in flight.  k=8 H=2048:
// T=4096 28 us, 5.3 TB/s, T=256 6.1; H=7168: T=4096 110, 4.8 TB/s, T=16 5.8 (up to 256 threads
// with the token's whole row: 116 and 11.4).
template <int DT>
__global__ __launch_bounds__(PM_THREADS) void unpermute_kernel(const UnpermP p) {
  constexpr int N = kPiece<DT>;
  const uint32_t u = blockIdx.x * PM_THREADS + threadIdx.x, in = u / (uint32_t)p.pieces, c = u - in * p.pieces;
  const int64_t t = blockIdx.y * p.turn + in;
  if (in >= p.turn || t >= p.T) return;
  const int32_t* position = p.position + t * p.k;
  const float* weights = p.weights != nullptr ? p.weights + t * p.k : nullptr;
  if (p.H < N) {
    float sum = 0.f;
    for (int s = 0; s < p.k; ++s) {
      const int at = position[s];
      if (at < 0 || at >= p.R) continue;
      const float v = pm_one<DT>(p.rows, at * p.ldr + c);
      sum = weights != nullptr ? fmaf(v, weights[s], sum) : sum + v;
    }
    pm_store_one(p.y_dtype, p.out, t * p.H + c, sum);
    return;
  }
  const int i = min((int)c * N, p.H - N);
  float sum[N];
#pragma unroll
  for (int e = 0; e < N; ++e) sum[e] = 0.f;
  for (int s0 = 0; s0 < p.k; s0 += 8) {
    u32x4 b[8];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = s0 + j < p.k ? position[s0 + j] : -1;
      const bool kept = at >= 0 && at < p.R;
      b[j] = kept ? pm_load(reinterpret_cast<const char*>(p.rows) + (at * p.ldr + i) * (DT == CCQ_F32 ? 4 : 2))
                  : u32x4{0, 0, 0, 0};
      w[j] = !kept ? 0.f : weights != nullptr ? weights[s0 + j] : 1.f;  // (0 times the zeros above, whatever the weight)
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v[N];
      pm_floats<DT>(b[j], v);
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = fmaf(v[e], w[j], sum[e]);
    }
  }
  pm_store_floats(p.y_dtype, p.out, t * p.H + i, sum);
}

// WAVES waves on a token: each piece of dy is read once, multiplied into the
// token's rows' gradients and with the rows themselves; the products' sums are
// joined over the lanes at the end (always in the same order).  T=2048 k=8 H=7168 bf16
// 104 us, 4.8 TB/s.
template <int DT, int WAVES>
__global__ __launch_bounds__(PM_THREADS) void unpermute_grad_kernel(const UnpermP p) {
  constexpr int N = kPiece<DT>, TOKENS = PM_WAVES / WAVES;
  __shared__ float part[PM_WAVES][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * TOKENS + wave / WAVES;
  const bool there = t < p.T;
  const int c = (wave % WAVES) * 64 + lane;
  constexpr int64_t E = DT == CCQ_F32 ? 4 : 2;
  for (int s0 = 0; s0 < p.k; s0 += 8) {
    float sum[8], w[8];
    int at[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum[j] = 0.f;
      const bool slot = there && s0 + j < p.k;
      at[j] = slot ? p.position[t * p.k + s0 + j] : INT32_MIN;
      w[j] = slot ? p.weights[t * p.k + s0 + j] : 0.f;
    }
    if (there) {
      if (p.H < N) {
        if (c < p.H) {
          const float g = pm_one<DT>(p.dy, t * p.ldy + c);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int row = at[j] < 0 ? ~at[j] : at[j];
            if (row >= p.R) continue;
            if (at[j] >= 0) sum[j] = pm_one<DT>(p.rows, row * p.ldr + c) * g;
            pm_store_one(DT, p.out, (int64_t)row * p.H + c, at[j] >= 0 ? w[j] * g : 0.f);
          }
        }
      } else {
        for (int h = c * N; h < p.H; h += WAVES * 64 * N) {
          const int i = min(h, p.H - N);
          const u32x4 gb = pm_load(reinterpret_cast<const char*>(p.dy) + (t * p.ldy + i) * E);
          u32x4 rb[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            rb[j] = at[j] >= 0 && at[j] < p.R ? pm_load(reinterpret_cast<const char*>(p.rows) + (at[j] * p.ldr + i) * E)
                                              : u32x4{0, 0, 0, 0};
          float g[N];
          pm_floats<DT>(gb, g);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int row = at[j] < 0 ? ~at[j] : at[j];
            if (row >= p.R) continue;
            float r[N], o[N];
            pm_floats<DT>(rb[j], r);
#pragma unroll
            for (int e = 0; e < N; ++e) {
              o[e] = at[j] >= 0 ? w[j] * g[e] : 0.f;
              // (a row's last piece counts what the piece before it does not have)
              if (at[j] >= 0 && e >= h - i) sum[j] = fmaf(r[e], g[e], sum[j]);
            }
            pm_store_floats(DT, p.out, (int64_t)row * p.H + i, o);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int m = 32; m; m >>= 1) sum[j] += wave_shfl_xor(sum[j], m);
    if constexpr (WAVES > 1) {
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[wave][j] = sum[j];
      __syncthreads();
      if (wave % WAVES == 0)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int v = 1; v < WAVES; ++v) sum[j] += part[wave + v][j];
      __syncthreads();
    }
    if (there && c == 0)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (s0 + j < p.k) p.d_weights[t * p.k + s0 + j] = sum[j];
  }
}

int64_t esize(int dt) { return dt == CCQ_F32 ? 4 : 2; }

int check_sizes(const char* what, const ccq_moe_permute_args& a) {
  CCQ_REQUIRE(a.dtype == CCQ_F32 || a.dtype == CCQ_F16 || a.dtype == CCQ_BF16, "%s: dtype %d", what, a.dtype);
  CCQ_REQUIRE(a.k >= 1 && a.k <= PM_MAX_K, "%s: k=%lld, 1 to %d", what, (long long)a.k, PM_MAX_K);
  CCQ_REQUIRE(a.T >= 0 && a.T <= PM_MAX_N && a.T * a.k <= PM_MAX_N,
              "%s: T=%lld tokens of %lld experts: at most 2^20 in all", what, (long long)a.T, (long long)a.k);
  CCQ_REQUIRE(a.H >= 1 && a.H <= 1 << 20, "%s: H=%lld, 1 to 2^20", what, (long long)a.H);
  return 0;
}

// tokens of a workgroup.  Ranking among all: 1, but 2 of more than 1024 tokens (T=16 k=8
// 4.9 us, by twos 6.4; T=2048 k=1 H=64 8.4 and 6.8, by fours 7.0).  By chunks: what
// makes a row's copy worth a workgroup, 4 KiB, up to 8 (T=65536 k=8, of 1, 2, 4, 8: H=64 98,
// 62, 44, 35 us; H=256 142, 99, 86, 72; H=512 193, 156, 140, 141; H=1024 292, 254, 264, 262;
// H=2048 498, 511, 504, 518).
void plan_permute(PermP& p, int64_t T, int64_t k, int64_t bytes) {
  p.n = (int)(T * k);
  p.tokens = p.n <= PM_SELF ? (T > 1024 ? 2 : 1) : (int)std::clamp<int64_t>(4096 / bytes, 1, 8);
  while (p.tokens * k > PM_OWN) p.tokens /= 2;
  p.chunks = (int)cdiv(p.n, PM_CHUNK);
}

}  // namespace

}  // namespace ccq

using namespace ccq;

extern "C" size_t ccq_moe_permute_workspace_size(int64_t T, int64_t k, int64_t num_experts) {
  if (T < 1 || T > PM_MAX_N || k < 1 || k > PM_MAX_K || num_experts < 1 || num_experts > PM_MAX_E ||
      T * k > PM_MAX_N || T * k <= PM_SELF)
    return 0;
  return (size_t)(cdiv(T * k, PM_CHUNK) + 1) * (num_experts + 1) * 4;
}

extern "C" int ccq_moe_permute(const ccq_moe_permute_args* args) {
  const char* what = "ccq_moe_permute";
  CCQ_REQUIRE(args != nullptr, "%s: null arguments", what);
  const ccq_moe_permute_args& a = *args;
  if (int rc = check_sizes(what, a)) return rc;
  CCQ_REQUIRE(a.num_experts >= 1 && a.num_experts <= PM_MAX_E, "%s: num_experts=%lld, 1 to %d", what,
              (long long)a.num_experts, PM_MAX_E);
  CCQ_REQUIRE(a.T <= 1 || a.ldx >= a.H, "%s: row stride %lld of rows of %lld", what, (long long)a.ldx, (long long)a.H);
  CCQ_REQUIRE(a.offsets != nullptr && (a.T == 0 || (a.x && a.ids && a.rows && a.position)), "%s: null pointer", what);
  const size_t e = (size_t)esize(a.dtype);
  CCQ_REQUIRE(aligned(a.x, e) && aligned(a.rows, e) && aligned(a.ids, 8) && aligned(a.position, 4) && aligned(a.offsets, 4),
              "%s: pointers must be aligned to their elements", what);
  const size_t need = ccq_moe_permute_workspace_size(a.T, a.k, a.num_experts);
  CCQ_REQUIRE(need == 0 || (a.workspace != nullptr && aligned(a.workspace, 16) && a.workspace_bytes >= need),
              "%s: workspace of %zu bytes needed", what, need);
  PermP p = {a.x, a.ids, a.rows, a.position, a.offsets, reinterpret_cast<int32_t*>(a.workspace), nullptr, a.ldx * (int64_t)e,
             a.T};
  plan_permute(p, a.T, a.k, a.H * (int64_t)e);
  p.k = (int)a.k;
  p.E = (int)a.num_experts;
  p.H = (int)a.H;
  p.esize = (int)e;
  const dim3 grid((uint32_t)(cdiv(a.T, p.tokens) + 1));
  const hipStream_t st = as_stream(a.stream);
  if (need) {
    p.total = p.table + (int64_t)p.chunks * (p.E + 1);
    launch(permute_rank_kernel, dim3((uint32_t)p.chunks), dim3(PM_THREADS), 0, st, p);
    if (int rc = launch_status(what)) return rc;
    launch(permute_scan_kernel, dim3((uint32_t)cdiv(p.E + 1, 64)), dim3(64 * PM_SCAN_WAVES), 0, st, p);
    if (int rc = launch_status(what)) return rc;
    launch(permute_copy_kernel, grid, dim3(PM_THREADS), 0, st, p);
  } else {
    launch(permute_kernel, grid, dim3(PM_THREADS), 0, st, p);
  }
  return launch_status(what);
}

extern "C" int ccq_moe_unpermute(const ccq_moe_permute_args* args) {
  const char* what = "ccq_moe_unpermute";
  CCQ_REQUIRE(args != nullptr, "%s: null arguments", what);
  const ccq_moe_permute_args& a = *args;
  if (int rc = check_sizes(what, a)) return rc;
  CCQ_REQUIRE(a.y_dtype == CCQ_F32 || a.y_dtype == CCQ_F16 || a.y_dtype == CCQ_BF16, "%s: y_dtype %d", what, a.y_dtype);
  CCQ_REQUIRE(a.T * a.k <= 1 || a.ldr >= a.H, "%s: row stride %lld of rows of %lld", what, (long long)a.ldr, (long long)a.H);
  if (a.T == 0) return 0;
  CCQ_REQUIRE(a.rows && a.position && a.y, "%s: null pointer", what);
  CCQ_REQUIRE(aligned(a.rows, (size_t)esize(a.dtype)) && aligned(a.position, 4) && aligned(a.weights, 4) &&
                  aligned(a.y, (size_t)esize(a.y_dtype)),
              "%s: pointers must be aligned to their elements", what);
  const int64_t piece = a.dtype == CCQ_F32 ? 4 : 8, pieces = a.H < piece ? a.H : cdiv(a.H, piece);
  const int64_t turn = imin64(a.T, (1ll << 30) / pieces);  // (so that a thread's number has 32 bits)
  const UnpermP p = {a.rows, a.position, a.weights, nullptr, a.y, nullptr, a.ldr, 0, a.T * a.k, a.T, (int)a.k, (int)a.H,
                     a.y_dtype, (int)pieces, turn};
  const dim3 grid((uint32_t)cdiv(turn * pieces, PM_THREADS), (uint32_t)cdiv(a.T, turn));
  const hipStream_t st = as_stream(a.stream);
  if (a.dtype == CCQ_BF16)
    launch(unpermute_kernel<CCQ_BF16>, grid, dim3(PM_THREADS), 0, st, p);
  else if (a.dtype == CCQ_F16)
    launch(unpermute_kernel<CCQ_F16>, grid, dim3(PM_THREADS), 0, st, p);
  else
    launch(unpermute_kernel<CCQ_F32>, grid, dim3(PM_THREADS), 0, st, p);
  return launch_status(what);
}

namespace ccq {
namespace {
template <int WAVES>
void launch_grad(int dtype, const UnpermP& p, hipStream_t st) {
  const dim3 grid((uint32_t)cdiv(p.T, PM_WAVES / WAVES));
  if (dtype == CCQ_BF16)
    launch(unpermute_grad_kernel<CCQ_BF16, WAVES>, grid, dim3(PM_THREADS), 0, st, p);
  else if (dtype == CCQ_F16)
    launch(unpermute_grad_kernel<CCQ_F16, WAVES>, grid, dim3(PM_THREADS), 0, st, p);
  else
    launch(unpermute_grad_kernel<CCQ_F32, WAVES>, grid, dim3(PM_THREADS), 0, st, p);
}
}  // namespace
}  // namespace ccq

extern "C" int ccq_moe_unpermute_grad(const ccq_moe_permute_args* args) {
  const char* what = "ccq_moe_unpermute_grad";
  CCQ_REQUIRE(args != nullptr, "%s: null arguments", what);
  const ccq_moe_permute_args& a = *args;
  if (int rc = check_sizes(what, a)) return rc;
  CCQ_REQUIRE((a.T * a.k <= 1 || a.ldr >= a.H) && (a.T <= 1 || a.ldx >= a.H), "%s: row strides %lld and %lld of rows of %lld",
              what, (long long)a.ldr, (long long)a.ldx, (long long)a.H);
  if (a.T == 0) return 0;
  CCQ_REQUIRE(a.x && a.rows && a.position && a.weights && a.y && a.d_weights, "%s: null pointer", what);
  const size_t e = (size_t)esize(a.dtype);
  CCQ_REQUIRE(aligned(a.x, e) && aligned(a.rows, e) && aligned(a.y, e) && aligned(a.position, 4) && aligned(a.weights, 4) &&
                  aligned(a.d_weights, 4),
              "%s: pointers must be aligned to their elements", what);
  const UnpermP p = {a.rows, a.position, a.weights, a.x, a.y, a.d_weights, a.ldr, a.ldx, a.T * a.k, a.T, (int)a.k, (int)a.H,
                     a.dtype, 0, 0};
  // a wave a token leaves no exchange at the end, four share the latency of a small batch (k=8 H=7168: T=16 27 us, by
  // fours 11; T=512 34 and 24; T=1024 47 and 46; T=2048 105 and 111; k=2 H=4096: T=1024 12.2 and 11.6; T=1536 13.9 and 15.4)
  if (a.T >= 1536)
    launch_grad<1>(a.dtype, p, as_stream(a.stream));
  else
    launch_grad<4>(a.dtype, p, as_stream(a.stream));
  return launch_status(what);
}
