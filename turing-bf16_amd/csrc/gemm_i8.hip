// Linears in 8-bit integers: x quantised per row (token), W per row (output channel), the
// products summed in int32, the two scales and the bias applied in fp32, one rounding to bf16.
//
//   sx[m] = max_k |x[m, k]| / 127      qx[m, k] = rint(127 x[m, k] / max_k |x[m, k]|)
//   y[m, n] = (sum_k qx[m, k] qw[n, k]) sx[m] sw[n] + b[n]
#include <algorithm>

#include "abi_util.h"
#include "common.h"

using namespace tbf16;

namespace {

typedef int int4i __attribute__((ext_vector_type(4)));

// ---- quantisation ---------------------------------------------------------------------

// What turns a row's values into codes. The code of x is rint(127 x / a), a = max |x|, ties
// to even, of the exact quotient. All in fp32: x and a are bf16 (8 bits), both multiplied by
// the power of two that brings a near 1 (c = 127 x 2^k is exact, 15 bits; where 2^k has to
// stop at 2^+-120 nothing overflows, and what underflows has code 0). With r = 1 / (a 2^k),
// p = c r is off by 2 roundings, its error e = c - p (a 2^k) comes from one fma, and p + e r
// is the quotient to one rounding. Quotients that are exactly n + 1/2 come out so; every
// other is off n + 1/2 by 2^-16 of itself at least (254 X 2^i - (2 n + 1) A is a nonzero
// integer, X and A the 8-bit significands), so no rounding carries one over a border.
struct RowCode {
  float mul, a, r;
};
__device__ __forceinline__ RowCode row_code(float amax) {
  const int k = min(max(-frexp_exp(amax), -120), 120);
  RowCode c;
  c.mul = 127.f * pow2f(k);
  c.a = amax * pow2f(k);
  c.r = amax > 0.f ? 1.f / c.a : 0.f;
  return c;
}
// The code in the low byte (two's complement): adding 1.5 x 2^23 rounds to an integer.
__device__ __forceinline__ uint32_t code_of(float x, const RowCode& rc) {
  const float c = x * rc.mul, p = c * rc.r;
  return __float_as_uint(fmaf(fmaf(-p, rc.a, c), rc.r, p) + 12582912.f);
}

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, kWave));
  return v;
}

// One wave per row. Rows whose maximum is not finite (an infinity or a NaN among their
// values: integers hold neither) get zero codes and a NaN scale, so every product with
// them is NaN.
__global__ __launch_bounds__(256) void quantize_rows_i8_kernel(const uint16_t* __restrict__ x, int64_t R, int64_t K,
                                                               int64_t ldx, uint8_t* __restrict__ y, int64_t ldy,
                                                               float* __restrict__ scale) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= R) return;
  const uint16_t* xr = x + row * ldx;
  uint32_t bits = 0;
  for (int64_t i = lane; i < K; i += 64) bits = max(bits, (uint32_t)xr[i] & 0x7fffu);
  bits = wave_max_u(bits);
  const bool finite = bits < 0x7f80u;
  const float amax = finite ? __uint_as_float(bits << 16) : 0.f;
  const RowCode rc = row_code(amax);
  for (int64_t i = lane; i < (K + 15) / 16 * 16; i += 64)
    y[row * ldy + i] = i < K && finite ? (uint8_t)code_of(bf16_lo(xr[i]), rc) : (uint8_t)0;
  if (lane == 0) scale[row] = finite ? amax / 127.f : NAN;
}

// ---- product ----------------------------------------------------------------------------

// One wave per 16 x 16 outputs, fragments straight from memory: lane l holds 16 codes of
// row l % 16, k = 16 (l / 16) of a 64-wide step.
__global__ __launch_bounds__(64) void gemm_i8_kernel(const uint8_t* __restrict__ A, int64_t lda,
                                                     const float* __restrict__ sa, const uint8_t* __restrict__ B,
                                                     int64_t ldb, const float* __restrict__ sb,
                                                     const uint16_t* __restrict__ bias, uint16_t* __restrict__ C,
                                                     int64_t ldc, int M, int N, int K16) {
  const int tiles_n = (N + 15) / 16;
  const int m0 = blockIdx.x / tiles_n * 16, n0 = blockIdx.x % tiles_n * 16;
  const int lane = threadIdx.x, fr = lane & 15, fk = lane >> 4;
  const uint8_t* ar = A + (int64_t)min(m0 + fr, M - 1) * lda;
  const uint8_t* br = B + (int64_t)min(n0 + fr, N - 1) * ldb;
  int4i acc = {0, 0, 0, 0};
  for (int k = 0; k < K16; k += 64) {
    const int kk = k + 16 * fk;
    int4i a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (kk < K16) {
      a = *reinterpret_cast<const int4i*>(ar + kk);
      b = *reinterpret_cast<const int4i*>(br + kk);
    }
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, acc, 0, 0, 0);
  }
  const int m = m0 + fr;
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + 4 * fk + i;
    if (m < M && n < N) {
      const float y = (float)acc[i] * (sa[m] * 0x1p-24f) * (sb[n] * 0x1p24f) + (bias ? bf16_lo(bias[n]) : 0.f);
      C[(int64_t)m * ldc + n] = (uint16_t)pack_bf16(y, 0.f);
    }
  }
}

int launch_quantize_i8(const void* x, int64_t R, int64_t K, int64_t ldx, void* y8, int64_t ldy, float* scale,
                       hipStream_t st) {
  quantize_rows_i8_kernel<<<(unsigned)cdiv(R, 4), 256, 0, st>>>((const uint16_t*)x, R, K, ldx, (uint8_t*)y8, ldy, scale);
  TB_LAUNCH_CHECK("quantize_rows_i8");
  return 0;
}

int check_rows_i8(const char* fn, const void* x, int64_t R, int64_t K, int64_t ldx) {
  TB_CHECK(R >= 0 && K >= 0 && R < (int64_t)1 << 31 && K <= TBF16_I8_MAX_K, "%s: bad shape (K at most %d)", fn,
           TBF16_I8_MAX_K);
  TB_CHECK(ldx >= K && (reinterpret_cast<uintptr_t>(x) & 1) == 0, "%s: bad row stride or alignment of x", fn);
  return 0;
}

struct LinearI8Ws {
  size_t scale, x8, bytes;
};
LinearI8Ws linear_i8_ws(int64_t M, int64_t K, int64_t N) {
  LinearI8Ws w{0, align_up((size_t)M * 4, 256), 0};
  w.bytes = align_up(w.x8 + (size_t)M * align_up((size_t)K, 16), 256);
  return w;
}

}  // namespace

extern "C" int tbf16_quantize_rows_i8(const void* x, int64_t R, int64_t K, int64_t ldx, void* y8, int64_t ldy, float* scale,
                                      void* stream) {
  if (int rc = check_rows_i8("quantize_rows_i8", x, R, K, ldx)) return rc;
  TB_CHECK(aligned16(y8) && ldy % 16 == 0 && ldy >= (int64_t)align_up((size_t)K, 16) && aligned4(scale),
           "quantize_rows_i8: rows of codes must be 16-byte aligned and padded to 16");
  if (R == 0) return 0;
  return launch_quantize_i8(x, R, K, ldx, y8, ldy, scale, as_stream(stream));
}

extern "C" size_t tbf16_linear_i8_ws_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K < 0 || N <= 0) return 0;
  return linear_i8_ws(M, K, N).bytes;
}

extern "C" int tbf16_linear_i8(const void* x, int64_t M, int64_t K, int64_t ldx, const void* w8, int64_t N, int64_t ldw,
                               const float* ws, const void* bias, void* y, int64_t ldy, void* workspace, int64_t ws_bytes,
                               void* stream) {
  if (int rc = check_rows_i8("linear_i8", x, M, K, ldx)) return rc;
  const int64_t K16 = (int64_t)align_up((size_t)K, 16);
  TB_CHECK(N >= 0 && N < (int64_t)1 << 31, "linear_i8: bad shape");
  TB_CHECK(aligned16(w8) && ldw % 16 == 0 && ldw >= K16 && ldw < (int64_t)1 << 23,
           "linear_i8: weight rows must be 16-byte aligned and padded to 16");
  TB_CHECK(aligned16(y) && ldy % 8 == 0 && ldy >= (int64_t)align_up((size_t)N, 8),
           "linear_i8: rows of y must be 16-byte aligned and padded to 8");
  TB_CHECK(aligned4(ws) && (reinterpret_cast<uintptr_t>(bias) & 1) == 0, "linear_i8: scales or bias misaligned");
  if (M == 0 || N == 0) return 0;
  const LinearI8Ws w = linear_i8_ws(M, K, N);
  TB_CHECK(aligned16(workspace) && workspace != nullptr, "linear_i8: workspace missing or misaligned");
  if (ws_bytes < (int64_t)w.bytes) {
    set_error("linear_i8: workspace too small (%lld bytes, needs %zu)", (long long)ws_bytes, w.bytes);
    return TBF16_EWS;
  }
  const hipStream_t st = as_stream(stream);
  uint8_t* wsp = static_cast<uint8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(wsp + w.scale);
  if (int rc = launch_quantize_i8(x, M, K, ldx, wsp + w.x8, K16, sx, st)) return rc;
  const int64_t blocks = cdiv(M, 16) * cdiv(N, 16);
  TB_CHECK(blocks < (int64_t)1 << 31, "linear_i8: grid too large");
  gemm_i8_kernel<<<(unsigned)blocks, 64, 0, st>>>(wsp + w.x8, K16, sx, (const uint8_t*)w8, ldw, ws, (const uint16_t*)bias,
                                                  (uint16_t*)y, ldy, (int)M, (int)N, (int)K16);
  TB_LAUNCH_CHECK("linear_i8");
  return 0;
}
