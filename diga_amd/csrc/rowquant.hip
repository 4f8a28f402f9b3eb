// Rows held in 8 bits: the producers of diga_matmul_fp8's left operand (no reference call site).
//   diga_rms_norm_fp8    h = x (+ r);  y = h * w / sqrt(mean(h^2) + eps)
//   diga_silu_mul_fp8    y = g / (1 + exp(-g)) * u,  x = [g | u]
//   diga_quantize_fp8    y = x
// and for every row and block of 128 columns   s = max(max|y|, 2^-100) / 448,   q = e4m3(y * (1 / s)), nearest even.
// All arithmetic is fp32; the roundings are q (the operator's output type) and h in x's type (the residual stream keeps
// the model's type; the norm itself is taken from the unrounded fp32 sum).  1 / s is one division per block of 128: the
// product y * (1 / s) is within 1.5 fp32 steps of y / s, i.e. a value changes its e4m3 neighbour only within 2^-22 of a tie.
// A NaN stays at its place (max ignores it); an infinite y makes its block's finite values 0 and itself NaN.
//
// Layout: a group of 16 lanes owns a block of 128 columns, 8 consecutive ones per lane, so the block's maximum is four lane exchanges
// and the block's scale one 4-byte store.  A lane's 8 values are one load (two for fp32) whatever the rows' alignment: the loads and
// stores are typed with the element's alignment, which the hardware takes; only a lane that crosses the row's end goes by elements.
#include "common.h"
#include <algorithm>

namespace {

constexpr float E4M3_MAX = 448.f;
constexpr float LEAST_AMAX = 7.888609052210118e-31f;      // 2^-100: the scale of an empty block stays a normal number

struct RowQuantParams {
  const void* x;
  const void* res;
  const void* weight;
  uint8_t* q;
  float* scale;
  void* h;
  int64_t M, ldx, ldr, ldq, ldh, ssm, ssb;
  int N, nb, wtype, up;             // up: column of the second half of a gated row
  float eps;
};

// lane j's 8 values of the block that starts at column c0; columns >= N read as 0
template <typename T>
struct Eight {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c0, int j, int N, float* v) {
  const int c = c0 + 8 * j;
  if (c + 8 <= N) {
    const typename Eight<T>::type a = *reinterpret_cast<const typename Eight<T>::type*>(row + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < N ? (float)row[c + e] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int c0, int j, int N, const float* v) {
  const int c = c0 + 8 * j;
  if (c + 8 <= N) {
    typename Eight<T>::type a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (T)v[e];
    *reinterpret_cast<typename Eight<T>::type*>(row + c) = a;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < N) row[c + e] = (T)v[e];
  }
}
__device__ __forceinline__ void load_weight8(const void* w, int wtype, int c0, int j, int N, float* v) {
  if (wtype == DIGA_BF16) load8(static_cast<const __bf16*>(w), c0, j, N, v);
  else if (wtype == DIGA_FP16) load8(static_cast<const _Float16*>(w), c0, j, N, v);
  else load8(static_cast<const float*>(w), c0, j, N, v);
}

// maximum of |y| over the 16 lanes of a block, then scale and the 8 e4m3 values of this lane
__device__ __forceinline__ void quantise8(const float* y, uint8_t* qrow, float* scale, int c0, int j, int N) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(y[e]));
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  m = fmaxf(m, LEAST_AMAX);
  const float s = m / E4M3_MAX, inv = 1.f / s;
  if (j == 0 && c0 < N) *scale = s;
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
  const int c = c0 + 8 * j;
  if (c + 8 <= N) {
    typedef unsigned int bytes8 __attribute__((ext_vector_type(2), aligned(1)));
    *reinterpret_cast<bytes8*>(qrow + c) = bytes8{(unsigned)lo, (unsigned)hi};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < N) qrow[c + e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
  }
}

// WPR waves share a row, CH blocks of 4 x 128 columns per wave: the row stays in registers (WPR * CH * 512 columns at most).  h may be
// written over x or the residual (a lane stores what it has read).  Bound by memory: many waves with one block each beat fewer with
// more loads in flight (8385 x 2048 bf16 with residual, 7 bytes per value: 22.5 us = 5.4 TB/s; measured when chosen, before loads
// of 16 bytes at any alignment: 4 waves x 1 block 26.7, 2 x 2 28.2, 1 x 4 30.6; weights loaded ahead of the sum 28.6 / 30.5 / 35.5).
template <typename T, int WPR, int CH>
__global__ __launch_bounds__(WPR < 4 ? 256 : WPR * 64) void rms_norm_fp8_kernel(RowQuantParams p) {
  constexpr int RPB = WPR < 4 ? 4 / WPR : 1;               // rows per block
  __shared__ float part[WPR * RPB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15;
  const int64_t m = (int64_t)blockIdx.x * RPB + wave / WPR;
  const int cw = (wave % WPR) * 512 + (lane >> 4) * 128;   // first column of this lane's first block
  const bool live = m < p.M;
  float h[CH][8], ss = 0.f;
  if (live) {
    const T* xr = static_cast<const T*>(p.x) + m * p.ldx;
#pragma unroll
    for (int i = 0; i < CH; ++i) load8(xr, cw + i * WPR * 512, j, p.N, h[i]);
    if (p.res) {
      const T* rr = static_cast<const T*>(p.res) + m * p.ldr;
      T* hr = static_cast<T*>(p.h) + m * p.ldh;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float r[8];
        load8(rr, cw + i * WPR * 512, j, p.N, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] += r[e];
        store8(hr, cw + i * WPR * 512, j, p.N, h[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) ss += __shfl_xor(ss, d);
  if constexpr (WPR > 1) {
    if (lane == 0) part[wave] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int v = 0; v < WPR; ++v) ss += part[(wave / WPR) * WPR + v];
  }
  if (!live) return;
  const float r = 1.f / sqrtf(ss / (float)p.N + p.eps);
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c0 = cw + i * WPR * 512;
    if (c0 >= p.N) continue;                               // the block's 16 lanes agree
    float w[8];
    load_weight8(p.weight, p.wtype, c0, j, p.N, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = h[i][e] * r * w[e];
    quantise8(w, p.q + m * p.ldq, p.scale + m * p.ssm + (int64_t)(c0 >> 7) * p.ssb, c0, j, p.N);
  }
}

// 16 groups of 16 lanes per block: 4 blocks of columns (fewer in narrow rows) by 4 or more rows, so that the scales of neighbouring
// rows leave together.  Bound by memory: 8385 x 4096 bf16, 5 bytes per value, 37.2 us = 4.6 TB/s (16 blocks of columns side by side
// 39.8, two rows per lane in flight 38.5, four 47.8).
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void act_fp8_kernel(RowQuantParams p, int gpr_log2) {
  const int grp = threadIdx.x >> 4, j = threadIdx.x & 15;
  const int b = blockIdx.x * (1 << gpr_log2) + (grp & ((1 << gpr_log2) - 1));
  const int64_t rpb = 16 >> gpr_log2;
  if (b >= p.nb) return;
  for (int64_t m = blockIdx.y * rpb + (grp >> gpr_log2); m < p.M; m += gridDim.y * rpb) {
    const T* xr = static_cast<const T*>(p.x) + m * p.ldx;
    float y[8];
    load8(xr, b * 128, j, p.N, y);
    if constexpr (GATED) {
      float u[8];
      load8(xr + p.up, b * 128, j, p.N, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] / (1.f + expf(-y[e])) * u[e];
    }
    quantise8(y, p.q + m * p.ldq, p.scale + m * p.ssm + b * p.ssb, b * 128, j, p.N);
  }
}

template <typename T>
void launch_rms(const RowQuantParams& p, hipStream_t s) {
  const int n = p.N;
#define DIGA_RMS(WPR, CH) \
  rms_norm_fp8_kernel<T, WPR, CH><<<dim3((unsigned)((p.M + (WPR < 4 ? 4 / WPR : 1) - 1) / (WPR < 4 ? 4 / WPR : 1))), WPR < 4 ? 256 : WPR * 64, 0, s>>>(p)
  if (n <= 512) DIGA_RMS(1, 1);
  else if (n <= 1024) DIGA_RMS(2, 1);
  else if (n <= 2048) DIGA_RMS(4, 1);
  else if (n <= 4096) DIGA_RMS(8, 1);
  else if (n <= 8192) DIGA_RMS(8, 2);
  else if (n <= 16384) DIGA_RMS(16, 2);
  else if (n <= 32768) DIGA_RMS(16, 4);
  else DIGA_RMS(16, 8);
#undef DIGA_RMS
}

constexpr int64_t MAX_ROWS = (int64_t)1 << 31, RMS_ROWS = (int64_t)1 << 21;

int check_rows(const char* who, const void* x, int64_t ldx, int type, int64_t M, int N, int64_t width, int max_n, const void* q, int64_t ldq, const float* scale) {
  DIGA_CHECK_ARG(M >= 0 && M < MAX_ROWS, "%s: M=%lld rows (0 .. 2^31 - 1)", who, (long long)M);
  DIGA_CHECK_ARG(N >= 1 && N <= max_n, "%s: N=%d columns (1 .. %d)", who, N, max_n);
  DIGA_CHECK_ARG(type == DIGA_BF16 || type == DIGA_FP16 || type == DIGA_FP32, "%s: unknown type %d", who, type);
  DIGA_CHECK_ARG(M == 0 || (x && q && scale), "%s: null pointer", who);
  DIGA_CHECK_ARG(M <= 1 || (ldx >= width && ldq >= N), "%s: row strides (%lld, %lld) below the row widths (%lld, %d)", who, (long long)ldx, (long long)ldq, (long long)width, N);
  return DIGA_OK;
}

int act_fp8(const char* who, bool gated, const void* x, int64_t ldx, int type, int64_t M, int N, void* q, int64_t ldq, float* scale,
            int64_t ssm, int64_t ssb, void* stream) {
  if (int rc = check_rows(who, x, ldx, type, M, N, gated ? 2ll * N : N, 1 << 24, q, ldq, scale)) return rc;
  if (M == 0) return DIGA_OK;
  RowQuantParams p{};
  p.x = x, p.q = static_cast<uint8_t*>(q), p.scale = scale;
  p.M = M, p.N = N, p.nb = cdiv(N, 128), p.ldx = ldx, p.ldq = ldq, p.ssm = ssm, p.ssb = ssb, p.up = gated ? N : 0;
  int g = 0;
  while (g < 2 && (1 << g) < p.nb) ++g;
  const int64_t rpb = 16 >> g;
  const dim3 grid(cdiv(p.nb, 1 << g), (unsigned)std::min<int64_t>((M + rpb - 1) / rpb, 65535));
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define DIGA_ACT(T)                                            \
  do {                                                         \
    if (gated) act_fp8_kernel<T, true><<<grid, 256, 0, s>>>(p, g); \
    else act_fp8_kernel<T, false><<<grid, 256, 0, s>>>(p, g);      \
  } while (0)
  if (type == DIGA_BF16) DIGA_ACT(__bf16);
  else if (type == DIGA_FP16) DIGA_ACT(_Float16);
  else DIGA_ACT(float);
#undef DIGA_ACT
  DIGA_CHECK_LAUNCH(who);
  return DIGA_OK;
}

}  // namespace

extern "C" int diga_rms_norm_fp8(const void* x, int64_t ldx, const void* residual, int64_t ldr, int type, const void* weight, int weight_type,
                                 float eps, int64_t M, int N, void* q, int64_t ldq, float* scale, int64_t scale_stride_m,
                                 int64_t scale_stride_b, void* residual_out, int64_t ldh, void* stream) {
  if (int rc = check_rows("diga_rms_norm_fp8", x, ldx, type, M, N, N, DIGA_RMS_NORM_MAX_N, q, ldq, scale)) return rc;
  DIGA_CHECK_ARG(weight_type == DIGA_BF16 || weight_type == DIGA_FP16 || weight_type == DIGA_FP32, "diga_rms_norm_fp8: unknown weight type %d", weight_type);
  DIGA_CHECK_ARG((residual == nullptr) == (residual_out == nullptr), "diga_rms_norm_fp8: residual and residual_out go together");
  DIGA_CHECK_ARG(M <= 1 || !residual || (ldr >= N && ldh >= N), "diga_rms_norm_fp8: row strides (%lld, %lld) below N=%d", (long long)ldr, (long long)ldh, N);
  DIGA_CHECK_ARG(eps >= 0.f, "diga_rms_norm_fp8: eps must not be negative");
  if (M == 0) return DIGA_OK;
  DIGA_CHECK_ARG(weight, "diga_rms_norm_fp8: null pointer");
  const int64_t size = type == DIGA_FP32 ? 4 : 2, wsize = weight_type == DIGA_FP32 ? 4 : 2;
  if (residual) {                                          // x or the residual itself may take the sum, nothing that lies across them
    const bool on_x = residual_out == x && (M == 1 || ldh == ldx), on_res = residual_out == residual && (M == 1 || ldh == ldr);
    DIGA_CHECK_ARG((on_x || !rows_meet(residual_out, M, ldh * size, N * size, x, M, ldx * size, N * size)) &&
                       (on_res || !rows_meet(residual_out, M, ldh * size, N * size, residual, M, ldr * size, N * size)) &&
                       !rows_meet(residual_out, M, ldh * size, N * size, weight, 1, 0, N * wsize),
                   "diga_rms_norm_fp8: residual_out lies across x, the residual or the weight");
  }
  RowQuantParams p{};
  p.x = x, p.res = residual, p.weight = weight, p.q = static_cast<uint8_t*>(q), p.scale = scale, p.h = residual_out;
  p.M = M, p.N = N, p.nb = cdiv(N, 128), p.ldx = ldx, p.ldr = ldr, p.ldq = ldq, p.ldh = ldh, p.ssm = scale_stride_m, p.ssb = scale_stride_b;
  p.wtype = weight_type, p.eps = eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t done = 0; done < M; done += RMS_ROWS) {     // a launch has fewer than 2^32 threads, up to 1024 of them a row
    p.M = std::min(M - done, RMS_ROWS);
    if (type == DIGA_BF16) launch_rms<__bf16>(p, s);
    else if (type == DIGA_FP16) launch_rms<_Float16>(p, s);
    else launch_rms<float>(p, s);
    DIGA_CHECK_LAUNCH("diga_rms_norm_fp8");
    p.x = static_cast<const char*>(p.x) + RMS_ROWS * ldx * size, p.q += RMS_ROWS * ldq, p.scale += RMS_ROWS * scale_stride_m;
    if (residual) p.res = static_cast<const char*>(p.res) + RMS_ROWS * ldr * size, p.h = static_cast<char*>(p.h) + RMS_ROWS * ldh * size;
  }
  return DIGA_OK;
}

extern "C" int diga_silu_mul_fp8(const void* x, int64_t ldx, int type, int64_t M, int N, void* q, int64_t ldq, float* scale,
                                 int64_t scale_stride_m, int64_t scale_stride_b, void* stream) {
  return act_fp8("diga_silu_mul_fp8", true, x, ldx, type, M, N, q, ldq, scale, scale_stride_m, scale_stride_b, stream);
}

extern "C" int diga_quantize_fp8(const void* x, int64_t ldx, int type, int64_t M, int N, void* q, int64_t ldq, float* scale,
                                 int64_t scale_stride_m, int64_t scale_stride_b, void* stream) {
  return act_fp8("diga_quantize_fp8", false, x, ldx, type, M, N, q, ldq, scale, scale_stride_m, scale_stride_b, stream);
}
