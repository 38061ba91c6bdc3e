// RMS norm of rows with the residual's addition and 8-bit output rows.
//
// Per row of H columns, in float32:
//   s = x + residual,  residual_out = round(s),
//   rstd = 1 / sqrt(mean(s^2) + eps),  p = s * w (one rounding),  y = round(p * rstd);
//   FP8 (a scale per 128 columns): m = max(max|p|, 1e-30),
//     q = e4m3(p * (448 / m)),  scale = m * rstd / 448;
//   INT8 (a scale per row): m = max(max|p|, 1e-30),
//     q = rint(p * (127 / m)) clamped to +-127,  scale = m * rstd / 127.
// rstd is common to the row, so it cancels out of p * rstd / scale: the codes
// are functions of p alone, do not move with the order of the row's sum, and
// the FP8 ones are stored before that sum is known.
//
// One pass.  Long batches are bound by HBM: 4096 rows of 7168 bf16 with a
// residual, FP8 and normalized rows move 265 MB in 48 us, 5.5 TB/s.  A few rows
// are one row's latency, 2.5 to 5 us.
#include "ccq_common.h"

#include <math.h>

namespace ccq {

namespace {

constexpr int64_t NORM_ROWS = 1 << 21;  // of a launch, which takes fewer than 2^32 threads (a second grid dimension
                                        // for the others costs each call 0.2 to 0.35 us)
constexpr float kNormTiny = 1e-30f;  // 127 or 448 over it is finite

struct NormP {
  const void* x;
  const void* residual;
  const void* w;
  void* residual_out;
  void* y;
  uint8_t* q;
  float* scale;
  int64_t ldx, ldr, ldo, rows;
  int H, w_dtype, y_dtype;
  float eps;
};

// 8 consecutive values of a row at any element alignment (one 16-byte access
// for 16-bit types, two for float32: the hardware takes unaligned ones), or
// the n < 8 that are left of it, the others 0.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, int n, float (&v)[8]) {
  if constexpr (DT == CCQ_F32) {
    const float* f = reinterpret_cast<const float*>(p) + i;
    if (n >= 8) {
      __builtin_memcpy(v, f, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? f[e] : 0.f;
    }
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + i;
    u32x4 b = {0, 0, 0, 0};
    if (n >= 8) {
      __builtin_memcpy(&b, h, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) b[e >> 1] |= (uint32_t)h[e] << (16 * (e & 1));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t u = (b[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
      v[e] = DT == CCQ_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, int n, const float (&v)[8]) {
  if constexpr (DT == CCQ_F32) {
    float* f = reinterpret_cast<float*>(p) + i;
    if (n >= 8) {
      __builtin_memcpy(f, v, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) f[e] = v[e];
    }
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p) + i;
    u32x4 b;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      b[e] = DT == CCQ_BF16 ? bf16x2_bits(v[2 * e], v[2 * e + 1])
                            : f32_to_f16_bits(v[2 * e]) | f32_to_f16_bits(v[2 * e + 1]) << 16;
    if (n >= 8) {
      __builtin_memcpy(h, &b, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) h[e] = (uint16_t)(b[e >> 1] >> (16 * (e & 1)));
    }
  }
}

__device__ __forceinline__ void load8_any(int dt, const void* p, int64_t i, int n, float (&v)[8]) {
  if (dt == CCQ_BF16)
    load8<CCQ_BF16>(p, i, n, v);
  else if (dt == CCQ_F16)
    load8<CCQ_F16>(p, i, n, v);
  else
    load8<CCQ_F32>(p, i, n, v);
}

__device__ __forceinline__ void store8_any(int dt, void* p, int64_t i, int n, const float (&v)[8]) {
  if (dt == CCQ_BF16)
    store8<CCQ_BF16>(p, i, n, v);
  else if (dt == CCQ_F16)
    store8<CCQ_F16>(p, i, n, v);
  else
    store8<CCQ_F32>(p, i, n, v);
}

// Columns 8 (t + THREADS i) .. + 7 of a row are vector i of its thread t; a
// row is held in registers, so x, residual and w are read once and HBM bounds
// long batches.  WAVES waves work on a row; one wave's workgroup takes four
// rows and needs no barrier.
template <int XT, int QF, int WAVES, int VPT>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void rms_norm_kernel(const NormP p) {
  constexpr int THREADS = 64 * WAVES;
  const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
  if (WAVES == 1 && row >= p.rows) return;
  float v[VPT][8], m[VPT];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = 8 * (t + THREADS * i), n = p.H - c;
    m[i] = 0.f;
    if (n > 0) {
      float w[8];
      load8<XT>(p.x, row * p.ldx + c, n, v[i]);
      if (p.residual != nullptr) {
        float r[8];
        load8<XT>(p.residual, row * p.ldr + c, n, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] += r[e];
      }
      load8_any(p.w_dtype, p.w, c, n, w);
      if (p.residual_out != nullptr) store8<XT>(p.residual_out, row * p.ldo + c, n, v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum = fmaf(v[i][e], v[i][e], sum);
        v[i][e] *= w[e];
        m[i] = fmaxf(m[i], fabsf(v[i][e]));
      }
    }
    if constexpr (QF == CCQ_Q_FP8_BLOCK) {  // 16 lanes hold a block of 128 columns
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) m[i] = fmaxf(m[i], __shfl_xor(m[i], off, 64));
      m[i] = fmaxf(m[i], kNormTiny);
      if (n > 0) {
        const float k = 448.0f / m[i];
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][0] * k, v[i][1] * k, 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][2] * k, v[i][3] * k, lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][4] * k, v[i][5] * k, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][6] * k, v[i][7] * k, hi, true);
        *reinterpret_cast<u32x2*>(p.q + row * p.H + c) = u32x2{(uint32_t)lo, (uint32_t)hi};
      }
    }
  }
  float mx = 0.f;
  if constexpr (QF == CCQ_Q_INT8_ROW) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) mx = fmaxf(mx, m[i]);
  }
  for (int off = 32; off >= 1; off >>= 1) {
    sum += __shfl_xor(sum, off, 64);
    if constexpr (QF == CCQ_Q_INT8_ROW) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  }
  if constexpr (WAVES > 1) {
    __shared__ float red[2][WAVES];
    if ((threadIdx.x & 63) == 0) {
      red[0][threadIdx.x >> 6] = sum;
      if constexpr (QF == CCQ_Q_INT8_ROW) red[1][threadIdx.x >> 6] = mx;
    }
    __syncthreads();
    sum = red[0][0];
    if constexpr (QF == CCQ_Q_INT8_ROW) mx = red[1][0];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) {
      sum += red[0][k];
      if constexpr (QF == CCQ_Q_INT8_ROW) mx = fmaxf(mx, red[1][k]);
    }
  }
  const float rstd = 1.0f / sqrtf(sum / (float)p.H + p.eps);
  float k127 = 0.f;
  if constexpr (QF == CCQ_Q_INT8_ROW) {
    mx = fmaxf(mx, kNormTiny);
    k127 = 127.0f / mx;
    if (t == 0) p.scale[row] = mx * rstd / 127.0f;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = 8 * (t + THREADS * i), n = p.H - c;
    if (n <= 0) break;
    if constexpr (QF == CCQ_Q_FP8_BLOCK) {
      if ((t & 15) == 0) p.scale[row * (p.H >> 7) + (c >> 7)] = m[i] * rstd / 448.0f;
    }
    if constexpr (QF == CCQ_Q_INT8_ROW) {
      uint32_t b[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q = rintf(v[i][e] * k127);
        const int z = q != q ? 0 : (int)fminf(fmaxf(q, -127.0f), 127.0f);  // a NaN's row has a NaN scale
        b[e >> 2] |= (uint32_t)(z & 255) << (8 * (e & 3));
      }
      uint8_t* q = p.q + row * p.H + c;
      if (n >= 8) {
        __builtin_memcpy(q, b, 8);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) q[e] = (uint8_t)(b[e >> 2] >> (8 * (e & 3)));
      }
    }
    if (p.y != nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= rstd;
      store8_any(p.y_dtype, p.y, row * p.H + c, n, v[i]);
    }
  }
}

// By the row's length, so that its threads hold one vector or two (four above
// 16384, where a workgroup has no more threads): longer chains of loads cost
// more than idle threads (GPU time in us, bf16 with a
// residual to FP8, 4096 rows; waves x vectors):
//   H = 512 1x1 5.8, 4x1 6.8; 1024 2x1 7.9, 4x1 9.1; 2048 4x1 14.8, 1x4 15.0;
//   7168 8x2 40.4 (5.1 TB/s), 16x1 42.4, 4x4 45.8; 2000 rows of 16384
//   16x2 45, 16x4 58.
// Up to 512 rows do not fill the CUs, and latency counts: one vector a thread
// (1 row of 4096 8x1 2.8, 4x2 3.7, 4096 rows 23.6 and 22.5; 1 row of 7168
// 16x1 3.4, 8x2 3.8, 4x4 5.8).
template <int XT, int QF>
int norm_launch(const NormP& p, hipStream_t st) {
  const dim3 one((unsigned)cdiv(p.rows, 4)), row((unsigned)p.rows);
  const bool few = p.rows <= 512;
  if (p.H <= 512)
    launch((rms_norm_kernel<XT, QF, 1, 1>), one, dim3(256), 0, st, p);
  else if (p.H <= 1024)
    launch((rms_norm_kernel<XT, QF, 2, 1>), row, dim3(128), 0, st, p);
  else if (p.H <= 2048)
    launch((rms_norm_kernel<XT, QF, 4, 1>), row, dim3(256), 0, st, p);
  else if (p.H <= 4096 && few)
    launch((rms_norm_kernel<XT, QF, 8, 1>), row, dim3(512), 0, st, p);
  else if (p.H <= 4096)
    launch((rms_norm_kernel<XT, QF, 4, 2>), row, dim3(256), 0, st, p);
  else if (p.H <= 8192 && few)
    launch((rms_norm_kernel<XT, QF, 16, 1>), row, dim3(1024), 0, st, p);
  else if (p.H <= 8192)
    launch((rms_norm_kernel<XT, QF, 8, 2>), row, dim3(512), 0, st, p);
  else if (p.H <= 16384)
    launch((rms_norm_kernel<XT, QF, 16, 2>), row, dim3(1024), 0, st, p);
  else
    launch((rms_norm_kernel<XT, QF, 16, 4>), row, dim3(1024), 0, st, p);
  return launch_status("ccq_rms_norm");
}

template <int XT>
int norm_dispatch(int q_fmt, const NormP& p, hipStream_t st) {
  if (q_fmt == CCQ_Q_FP8_BLOCK) return norm_launch<XT, CCQ_Q_FP8_BLOCK>(p, st);
  if (q_fmt == CCQ_Q_INT8_ROW) return norm_launch<XT, CCQ_Q_INT8_ROW>(p, st);
  return norm_launch<XT, CCQ_Q_NONE>(p, st);
}

bool is_float_code(int dt) { return dt == CCQ_F32 || dt == CCQ_F16 || dt == CCQ_BF16; }

}  // namespace

}  // namespace ccq

using namespace ccq;

extern "C" int ccq_rms_norm(const void* x, int x_dtype, int64_t ldx, const void* residual, int64_t ldr, const void* w,
                            int w_dtype, float eps, void* residual_out, int64_t ldo, void* y, int y_dtype, int q_fmt,
                            void* q, float* scale, int64_t rows, int64_t H, void* stream) {
  CCQ_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "ccq_rms_norm: rows=%lld outside [0, 2^31)", (long long)rows);
  CCQ_REQUIRE(H >= 1 && H <= 32768, "ccq_rms_norm: H=%lld outside [1, 32768]", (long long)H);
  CCQ_REQUIRE(is_float_code(x_dtype), "ccq_rms_norm: bad x_dtype");
  CCQ_REQUIRE(is_float_code(w_dtype), "ccq_rms_norm: bad w_dtype");
  CCQ_REQUIRE(y == nullptr || is_float_code(y_dtype), "ccq_rms_norm: bad y_dtype");
  CCQ_REQUIRE(q_fmt == CCQ_Q_NONE || q_fmt == CCQ_Q_FP8_BLOCK || q_fmt == CCQ_Q_INT8_ROW, "ccq_rms_norm: bad q_fmt");
  CCQ_REQUIRE(q_fmt != CCQ_Q_FP8_BLOCK || H % 128 == 0, "ccq_rms_norm: H=%lld not a multiple of 128 (FP8 blocks)",
              (long long)H);
  CCQ_REQUIRE(eps > 0.f && isfinite(eps), "ccq_rms_norm: eps must be positive and finite");
  CCQ_REQUIRE(ldx >= H && (residual == nullptr || ldr >= H) && (residual_out == nullptr || ldo >= H),
              "ccq_rms_norm: a row stride below H=%lld", (long long)H);
  if (rows == 0) return 0;
  CCQ_REQUIRE(x && w && (y || residual_out || q_fmt != CCQ_Q_NONE), "ccq_rms_norm: null pointer");
  CCQ_REQUIRE(q_fmt == CCQ_Q_NONE || (q && scale), "ccq_rms_norm: null pointer (q, scale)");
  const size_t e = x_dtype == CCQ_F32 ? 4 : 2;
  CCQ_REQUIRE(aligned(x, e) && aligned(residual, e) && aligned(residual_out, e) &&
                  aligned(w, w_dtype == CCQ_F32 ? 4 : 2) && aligned(y, y_dtype == CCQ_F32 ? 4 : 2) &&
                  aligned(scale, 4),
              "ccq_rms_norm: a pointer is not aligned to its elements");
  CCQ_REQUIRE(q_fmt != CCQ_Q_FP8_BLOCK || aligned(q, 8), "ccq_rms_norm: q must be 8-byte aligned");
  hipStream_t st = as_stream(stream);
  const size_t ye = y_dtype == CCQ_F32 ? 4 : 2;
  auto at = [](const void* b, int64_t i, size_t size) { return b == nullptr ? nullptr : (char*)b + i * size; };
  for (int64_t r = 0; r < rows; r += NORM_ROWS) {
    const NormP p = {at(x, r * ldx, e), at(residual, r * ldr, e), w, at(residual_out, r * ldo, e), at(y, r * H, ye),
                     (uint8_t*)at(q, r * H, 1), (float*)at(scale, r * (q_fmt == CCQ_Q_FP8_BLOCK ? H >> 7 : 1), 4),
                     ldx, ldr, ldo, rows - r < NORM_ROWS ? rows - r : NORM_ROWS, (int)H, w_dtype, y_dtype, eps};
    const int rc = x_dtype == CCQ_BF16  ? norm_dispatch<CCQ_BF16>(q_fmt, p, st)
                   : x_dtype == CCQ_F16 ? norm_dispatch<CCQ_F16>(q_fmt, p, st)
                                        : norm_dispatch<CCQ_F32>(q_fmt, p, st);
    if (rc) return rc;
  }
  return 0;
}

extern "C" int ccq_rms_norm_packed(const ccq_rms_norm_args* a) {
  CCQ_REQUIRE(a != nullptr, "ccq_rms_norm_packed: null arguments");
  return ccq_rms_norm(a->x, a->x_dtype, a->ldx, a->residual, a->ldr, a->w, a->w_dtype, a->eps, a->residual_out, a->ldo,
                      a->y, a->y_dtype, a->q_fmt, a->q, a->scale, a->rows, a->H, a->stream);
}
