// Linears in 8-bit integers: x quantised per row (token), W per row (output channel), the
// products summed in int32, the two scales and the bias applied in fp32, one rounding to bf16.
//
//   sx[m] = max_k |x[m, k]| / 127      qx[m, k] = rint(127 x[m, k] / max_k |x[m, k]|)
//   y[m, n] = (sum_k qx[m, k] qw[n, k]) sx[m] sw[n] + b[n]
#include <algorithm>

#include "abi_util.h"
#include "common.h"
#include "gemm_i8_plan.h"
#include "gemm_tiles.h"

using namespace tbf16;
using namespace tbf16::i8;

namespace {

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
// The larger magnitude's bits of two or eight bf16: as integers, so that a NaN counts as larger
// than an infinity and no value is lost.
__device__ __forceinline__ uint32_t mag2(uint32_t v) { return max(v & 0x7fffu, (v >> 16) & 0x7fffu); }
__device__ __forceinline__ uint32_t mag8(uint4 v) { return max(max(mag2(v.x), mag2(v.y)), max(mag2(v.z), mag2(v.w))); }
// The codes of two or eight bf16, packed.
__device__ __forceinline__ uint32_t codes4(uint32_t a, uint32_t b, const RowCode& rc) {
  const uint32_t lo = __builtin_amdgcn_perm(code_of(bf16_hi(a), rc), code_of(bf16_lo(a), rc), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code_of(bf16_hi(b), rc), code_of(bf16_lo(b), rc), 0x04000c0cu);
  return lo | hi;
}
__device__ __forceinline__ uint2 codes8(uint4 v, const RowCode& rc) {
  return make_uint2(codes4(v.x, v.y, rc), codes4(v.z, v.w, rc));
}
// Rows whose maximum is not finite (an infinity or a NaN among their values: integers hold
// neither) get zero codes and a NaN scale, so every product with them is NaN.
__device__ __forceinline__ float row_max(uint32_t bits) { return bits < 0x7f80u ? __uint_as_float(bits << 16) : 0.f; }
__device__ __forceinline__ float row_scale(uint32_t bits) {
  return bits < 0x7f80u ? __uint_as_float(bits << 16) / 127.f : NAN;
}

// TPR threads per row: a block of 4 waves (the row's latency is what a call of few rows waits for: 256 x
// 4096 6.2 us with a wave per row, 4.2 us so; 4096 x 4096, bound by memory: 12.4 and 11.1 us, 4.5 TB/s),
// or a wave where there are many rows of up to 2048 values (7363 x 448 with its product: 19.0 -> 14.2 us;
// 249 x 2040: 10.0 and, by waves, 10.7). VEC: rows of 16-byte chunks (K % 8 == 0), up to NC a
// thread held in registers between the maximum and the codes (one read of x), longer rows read
// twice; otherwise value by value. Codes are written up to Kp (zeros past K).
constexpr int kQThreads = 256;
template <bool VEC, int TPR, int NC>
__global__ __launch_bounds__(kQThreads) void quantize_rows_i8_kernel(const uint16_t* __restrict__ x, int R, int K,
                                                                     int64_t ldx, uint8_t* __restrict__ y, int64_t ldy,
                                                                     int Kp, float* __restrict__ scale) {
  __shared__ uint32_t amax[kQThreads / kWave];
  constexpr int ROWS = kQThreads / TPR;
  const int tid = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  if (ROWS > 1 && row >= R) return;
  const uint16_t* xr = x + row * ldx;
  uint8_t* yr = y + row * ldy;
  auto reduce = [&](uint32_t bits) {
    bits = wave_max_u(bits);
    if constexpr (ROWS == 1) {
      if ((tid & 63) == 0) amax[tid >> 6] = bits;
      __syncthreads();
      bits = max(max(amax[0], amax[1]), max(amax[2], amax[3]));
    }
    if (tid == 0) scale[row] = row_scale(bits);
    return bits;
  };
  uint32_t bits = 0;
  if constexpr (VEC) {
    const uint4* src = reinterpret_cast<const uint4*>(xr);
    uint2* dst = reinterpret_cast<uint2*>(yr);
    const int K8 = K >> 3, Kp8 = Kp >> 3;
    constexpr int STEP = TPR * NC;
    uint4 v[NC];
    auto load = [&](int i0) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int i = i0 + tid + c * TPR;
        v[c] = make_uint4(0, 0, 0, 0);
        if (i < K8) v[c] = src[i];
      }
    };
    for (int i = 0; i < K8; i += STEP) {
      load(i);
#pragma unroll
      for (int c = 0; c < NC; ++c) bits = max(bits, mag8(v[c]));
    }
    bits = reduce(bits);
    const RowCode rc = row_code(row_max(bits));
    for (int i0 = 0; i0 < Kp8; i0 += STEP) {
      if (Kp8 > STEP) load(i0);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int i = i0 + tid + c * TPR;
        if (i < Kp8) dst[i] = bits < 0x7f80u ? codes8(v[c], rc) : make_uint2(0, 0);
      }
    }
  } else {
    for (int i = tid; i < K; i += TPR) bits = max(bits, (uint32_t)xr[i] & 0x7fffu);
    bits = reduce(bits);
    const RowCode rc = row_code(row_max(bits));
    for (int i = tid; i < Kp; i += TPR)
      yr[i] = i < K && bits < 0x7f80u ? (uint8_t)code_of(bf16_lo(xr[i]), rc) : (uint8_t)0;
  }
}

// ---- product of few rows (decoding) -------------------------------------------------------
//
// At most 16 rows: the weight stream bounds it, N K bytes. A block of 8 waves owns R weight rows, as
// many as spread the weight over every CU (R <= 16 T; the rest of its last tile loads as zeros,
// without memory traffic). Its waves take K in turns of 128 bytes (two MFMAs of 64 a row),
// weights straight from memory into registers, PF turns of a wave in flight; the int32 sums of
// the waves meet in LDS. A lane's fragment is 16 bytes of weight row l % 16, and the same k of
// token l % 16.
// FUSED: every block quantises the tokens into LDS for itself, while its first weights are on their
// way: one launch, no workspace. 1: a single token (1 x 4096 x 4096: 6.4 us, 8.8 with a pass of its own;
// 1 x 32768 x 2048: 21 and 31). 3: 5 to 16 tokens of up to kFusedK values, two a wave, held in registers
// (8 x 4096 x 4096: 8.0 and 9.6; 16 x 2560 x 10240: 11.6 and 11.2, but 11 and 14 with the host's second
// launch). 2: 2 to 4 tokens of up to kFusedCodes values, two of four times that, read twice (4 x 4096
// x 4096: 8.1 and 9.0); above them the blocks' repeated work costs more than the pass (8 x 8192).
// 0: the codes come from a pass of their own (padded with zeros to a multiple of 128, so that what
// lies behind a weight row does not matter).
// 1 x 2560 x 10240 from HBM: 8.4 us, 3.1 TB/s of weights (6.4 where they are in the on-chip cache).
template <int T, int FUSED>
__global__ __launch_bounds__(512) void decode_i8_kernel(const uint16_t* __restrict__ x, int64_t ldx,
                                                        const uint8_t* __restrict__ x8, const float* __restrict__ sx,
                                                        const uint8_t* __restrict__ W, int64_t ldw,
                                                        const float* __restrict__ sw, const uint16_t* __restrict__ bias,
                                                        uint16_t* __restrict__ y, int64_t ldy, int M, int N, int K, int R) {
  constexpr int WAVES = 8, PF = T == 1 ? 8 : T == 2 ? 4 : 3;
  extern __shared__ __align__(16) uint8_t xl[];  // FUSED: [M][Kp + 16] codes
  __shared__ intx4 red[WAVES][T][64];
  __shared__ uint32_t amax[WAVES][kDecodeRows];
  __shared__ float scale[kDecodeRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * R, nend = min(N, n0 + R);
  const int turns = (K + 127) / 128, Kp = turns * 128;
  const BufRes wres = make_res(W + (int64_t)n0 * ldw, (int64_t)(nend - n0) * ldw);  // (below 2^29)
  int woff[T];
#pragma unroll
  for (int t = 0; t < T; ++t) woff[t] = (16 * t + fr) * (int)ldw + 16 * g;
  uint4 w[PF][T][2];
  auto load = [&](uint4 (&w)[T][2], int turn) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) w[t][s] = buf_load16(wres, woff[t] + 64 * s, turn * 128);
  };
#pragma unroll
  for (int u = 0; u < PF; ++u)
    if (wave + u * WAVES < turns) load(w[u], wave + u * WAVES);

  if constexpr (FUSED == 3) {
    // a wave takes tokens `wave` and `wave` + 8, all their chunks in registers
    const int K8 = K >> 3, Kp8 = Kp >> 3;
    constexpr int NC = kFusedK / 512;
    uint4 v[2][NC];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int m = wave + 8 * r;
      const uint4* src = reinterpret_cast<const uint4*>(x + m * ldx);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        v[r][c] = make_uint4(0, 0, 0, 0);
        if (m < M && 64 * c + lane < K8) v[r][c] = src[64 * c + lane];
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int m = wave + 8 * r;
      if (m >= M) break;
      uint32_t bits = 0;
#pragma unroll
      for (int c = 0; c < NC; ++c) bits = max(bits, mag8(v[r][c]));
      bits = wave_max_u(bits);
      const RowCode rc = row_code(row_max(bits));
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (64 * c + lane < Kp8)
          *reinterpret_cast<uint2*>(xl + m * (Kp + 16) + 8 * (64 * c + lane)) =
              bits < 0x7f80u ? codes8(v[r][c], rc) : make_uint2(0, 0);
      if (lane == 0) scale[m] = row_scale(bits);
    }
    __syncthreads();
  } else if constexpr (FUSED != 0) {
    const int K8 = K >> 3, Kp8 = Kp >> 3;
    // `per` waves on a row, 8 / per rows at once
    const int lg = FUSED == 1 ? 3 : M == 2 ? 2 : 1, per = 1 << lg;
    const int first = wave >> lg, part = wave & (per - 1), step = per * 64, i0 = part * 64 + lane;
    for (int m = first; m < (FUSED == 1 ? 1 : M); m += WAVES >> lg) {
      const uint4* src = reinterpret_cast<const uint4*>(x + m * ldx);
      uint32_t bits = 0;
#pragma unroll 4
      for (int i = i0; i < K8; i += step) bits = max(bits, mag8(src[i]));
      bits = wave_max_u(bits);
      if (lane == 0) amax[part][m] = bits;
    }
    __syncthreads();
    for (int m = first; m < (FUSED == 1 ? 1 : M); m += WAVES >> lg) {
      const uint4* src = reinterpret_cast<const uint4*>(x + m * ldx);
      uint32_t bits = amax[0][m];
#pragma unroll
      for (int i = 1; i < WAVES; ++i) bits = max(bits, i < per ? amax[i][m] : 0u);
      const RowCode rc = row_code(row_max(bits));
#pragma unroll 4
      for (int i = i0; i < Kp8; i += step) {
        uint2 c = make_uint2(0, 0);
        if (i < K8 && bits < 0x7f80u) c = codes8(src[i], rc);
        *reinterpret_cast<uint2*>(xl + m * (Kp + 16) + 8 * i) = c;
      }
      if (i0 == 0) scale[m] = row_scale(bits);
    }
    __syncthreads();
  }
  // tokens past M take the last one's codes and are not stored
  const int mr = FUSED == 1 ? 0 : min(fr, M - 1);
  const uint8_t* xr = (FUSED ? xl + mr * (Kp + 16) : x8 + (int64_t)mr * Kp) + 16 * g;
  intx4 acc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) acc[t] = intx4{0, 0, 0, 0};
  for (int t0 = wave; t0 < turns; t0 += PF * WAVES) {
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      const int turn = t0 + u * WAVES;
      if (turn >= turns) break;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const intx4 xf = *reinterpret_cast<const intx4*>(xr + turn * 128 + 64 * s);
#pragma unroll
        for (int t = 0; t < T; ++t) acc[t] = I8Op::mma(__builtin_bit_cast(intx4, w[u][t][s]), xf, acc[t]);
      }
      if (turn + PF * WAVES < turns) load(w[u], turn + PF * WAVES);
    }
  }
#pragma unroll
  for (int t = 0; t < T; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  if (tid >= T * 64) return;
  const int t = tid >> 6, m = lane & 15, n = n0 + 16 * t + 4 * g;
  if (m >= M || n >= (nend + 3) / 4 * 4) return;
  intx4 v = red[0][t][lane];
#pragma unroll
  for (int k = 1; k < WAVES; ++k) v += red[k][t][lane];
  const float sa = (FUSED ? scale[m] : sx[m]) * I8Op::kA;
  float f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = min(n + e, N - 1);
    f[e] = fmaf((float)v[e] * sa, sw[c] * I8Op::kB, bias ? bf16_lo(bias[c]) : 0.f);
  }
  *reinterpret_cast<uint2*>(y + (int64_t)m * ldy + n) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
}

// ---- product of many rows -------------------------------------------------------------------

// Split K: the sum of the tile kernels' int32 partial sums (splits x M x Np) and the epilogue.
// One thread per 8 columns of a row.
__global__ __launch_bounds__(256) void splitk_i8_kernel(const intx4* __restrict__ part, int splits,
                                                        const float* __restrict__ sx, const float* __restrict__ sw,
                                                        const uint16_t* __restrict__ bias, uint16_t* __restrict__ y,
                                                        int64_t ldy, int M, int N, int Np) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)M * (Np / 8)) return;
  const int m = (int)(i / (Np / 8)), n = (int)(i % (Np / 8)) * 8;
  const int64_t step = (int64_t)M * (Np / 4);
  intx4 lo = part[2 * i], hi = part[2 * i + 1];
  for (int k = 1; k < splits; ++k) {
    lo += part[2 * i + k * step];
    hi += part[2 * i + 1 + k * step];
  }
  const float sa = sx[m] * I8Op::kA;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = min(n + e, N - 1);
    f[e] = fmaf((float)(e < 4 ? lo[e & 3] : hi[e & 3]) * sa, sw[c] * I8Op::kB, bias ? bf16_lo(bias[c]) : 0.f);
  }
  stg16(y + (int64_t)m * ldy + n, make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]),
                                             pack_bf16(f[6], f[7])));
}

// The last plans of this thread by shape (the search costs as much host time as a launch).
const Plan& plan(int64_t M, int64_t K, int64_t N, bool vec) {
  struct Entry {
    int64_t M, K, N, cus;
    bool vec;
    Plan plan;
  };
  constexpr int kEntries = 64;
  static thread_local Entry cache[kEntries] = {};  // M = 0: empty
  Entry& e = cache[(uint64_t)(M * 31 + N * 7 + K) % kEntries];
  const int64_t cus = num_cus();
  if (e.M != M || e.K != K || e.N != N || e.cus != cus || e.vec != vec) e = Entry{M, K, N, cus, vec, plan_of(M, K, N, vec, cus)};
  return e.plan;
}

bool rows_vec(const void* x, int64_t K, int64_t ldx) { return K % 8 == 0 && ldx % 8 == 0 && aligned16(x); }

int launch_quantize_i8(const void* x, int64_t R, int64_t K, int64_t ldx, void* y8, int64_t ldy, int64_t Kp, float* scale,
                       hipStream_t st) {
  const bool vec = rows_vec(x, K, ldx), wave = K <= 2048 && R > num_cus();
  const unsigned blocks = (unsigned)(wave ? cdiv(R, kQThreads / kWave) : R);
#define QUANTIZE(VEC_, TPR_, NC_)                                                                                \
  quantize_rows_i8_kernel<VEC_, TPR_, NC_><<<blocks, kQThreads, 0, st>>>((const uint16_t*)x, (int)R, (int)K, ldx, (uint8_t*)y8, ldy, \
                                                                    (int)Kp, scale)
  if (vec) {
    if (wave) QUANTIZE(true, kWave, 4);
    else if (K <= 4096) QUANTIZE(true, kQThreads, 2);
    else QUANTIZE(true, kQThreads, 4);
  } else {
    if (wave) QUANTIZE(false, kWave, 1);
    else QUANTIZE(false, kQThreads, 1);
  }
#undef QUANTIZE
  TB_LAUNCH_CHECK("quantize_rows_i8");
  return 0;
}

int check_rows_i8(const char* fn, const void* x, int64_t R, int64_t K, int64_t ldx) {
  TB_CHECK(R >= 0 && K >= 0 && R < (int64_t)1 << 31 && K <= TBF16_I8_MAX_K, "%s: bad shape (K at most %d)", fn,
           TBF16_I8_MAX_K);
  TB_CHECK(ldx >= K && (reinterpret_cast<uintptr_t>(x) & 1) == 0, "%s: bad row stride or alignment of x", fn);
  return 0;
}

}  // namespace

extern "C" int tbf16_quantize_rows_i8(const void* x, int64_t R, int64_t K, int64_t ldx, void* y8, int64_t ldy, float* scale,
                                      void* stream) {
  if (int rc = check_rows_i8("quantize_rows_i8", x, R, K, ldx)) return rc;
  TB_CHECK(aligned16(y8) && ldy % 16 == 0 && ldy >= (int64_t)align_up((size_t)K, 16) && aligned4(scale),
           "quantize_rows_i8: rows of codes must be 16-byte aligned and padded to 16");
  if (R == 0) return 0;
  return launch_quantize_i8(x, R, K, ldx, y8, ldy, (int64_t)align_up((size_t)K, 16), scale, as_stream(stream));
}

extern "C" size_t tbf16_linear_i8_ws_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K < 0 || N <= 0) return 0;
  return plan(M, K, N, false).bytes;  // (enough for the forms that need none)
}

extern "C" int tbf16_linear_i8(const void* x, int64_t M, int64_t K, int64_t ldx, const void* w8, int64_t N, int64_t ldw,
                               const float* ws, const void* bias, void* y, int64_t ldy, void* workspace, int64_t ws_bytes,
                               void* stream) {
  if (int rc = check_rows_i8("linear_i8", x, M, K, ldx)) return rc;
  const int64_t K16 = (int64_t)align_up((size_t)K, 16), Np = (int64_t)align_up((size_t)N, 8);
  TB_CHECK(N >= 0 && N < ((int64_t)1 << 31) - 512 && M < ((int64_t)1 << 31) - 512, "linear_i8: bad shape");
  TB_CHECK(aligned16(w8) && ldw % 16 == 0 && ldw >= K16 && ldw < (int64_t)1 << 23,
           "linear_i8: weight rows must be 16-byte aligned and padded to 16");
  TB_CHECK(aligned16(y) && ldy % 8 == 0 && ldy >= Np, "linear_i8: rows of y must be 16-byte aligned and padded to 8");
  TB_CHECK(aligned4(ws) && (reinterpret_cast<uintptr_t>(bias) & 1) == 0, "linear_i8: scales or bias misaligned");
  if (M == 0 || N == 0) return 0;
  const Plan& p = plan(M, K, N, rows_vec(x, K, ldx));
  TB_CHECK(aligned16(workspace) && (workspace != nullptr || p.bytes == 0), "linear_i8: workspace missing or misaligned");
  if (ws_bytes < (int64_t)p.bytes) {
    set_error("linear_i8: workspace too small (%lld bytes, needs %zu)", (long long)ws_bytes, p.bytes);
    return TBF16_EWS;
  }
  const hipStream_t st = as_stream(stream);
  uint8_t* wsp = static_cast<uint8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(wsp + p.scale);
  uint8_t* x8 = wsp + p.x8;
  const int64_t Kp = (int64_t)align_up((size_t)K, 128);
  const uint16_t* bi = (const uint16_t*)bias;
  uint16_t* yo = (uint16_t*)y;
  if (!p.fused)
    if (int rc = launch_quantize_i8(x, M, K, ldx, x8, Kp, Kp, sx, st)) return rc;
  if (p.decode) {
    const unsigned blocks = (unsigned)cdiv(N, p.R);
#define DECODE(T_, FUSED_)                                                                                   \
  decode_i8_kernel<T_, FUSED_><<<blocks, 512, FUSED_ ? (size_t)(M * (Kp + 16)) : 0, st>>>(                   \
      (const uint16_t*)x, ldx, x8, sx, (const uint8_t*)w8, ldw, ws, bi, yo, ldy, (int)M, (int)N, (int)K, p.R)
#define DECODE_T(FUSED_)                \
  switch (p.T) {                        \
    case 1: DECODE(1, FUSED_); break;   \
    case 2: DECODE(2, FUSED_); break;   \
    case 3: DECODE(3, FUSED_); break;   \
    default: DECODE(4, FUSED_); break;  \
  }
    switch (p.fused) {
      case 0: DECODE_T(0) break;
      case 1: DECODE_T(1) break;
      case 2: DECODE_T(2) break;
      default: DECODE_T(3) break;
    }
#undef DECODE_T
#undef DECODE
    TB_LAUNCH_CHECK("linear_i8");
    return 0;
  }
  // operand rows in units of 2 bytes
  const auto a = (const uint16_t*)x8, b = (const uint16_t*)w8;
  const Tile& t = kTiles[p.tile];
  float* part = p.splits > 1 ? reinterpret_cast<float*>(wsp + p.part) : nullptr;
  const int kt_per = (int)cdiv(Kp / 128, p.splits);
  const dim3 grid((unsigned)(cdiv(M, t.bm) * cdiv(Np, p.rows)), (unsigned)p.splits);
#define PINGPONG(HA_, FB_, S_)                                                                                   \
  pingpong_kernel<I8Op, HA_, FB_, S_, true><<<grid, 512, 0, st>>>(a, Kp / 2, sx, b, ldw / 2, ws, bi, yo, ldy, (int)M, (int)Np, \
                                                                  (int)(Kp / 2), part, kt_per, (int)N)
#define KSPLIT(RM_, RN_, S_)                                                                                             \
  ksplit_kernel<I8Op, RM_, RN_, S_, true><<<grid, 512, 0, st>>>(a, Kp / 2, sx, b, ldw / 2, ws, bi, yo, ldy, (int)M, (int)Np, \
                                                                (int)(Kp / 2), part, kt_per, p.rows, (int)N, ConvGeom{})
  switch (p.tile) {
    case 0: PINGPONG(4, 2, 2); break;
    case 1: PINGPONG(3, 2, 2); break;
    case 2: PINGPONG(2, 2, 3); break;
    case 3: PINGPONG(4, 1, 3); break;
    case 4: KSPLIT(8, 4, 3); break;
    case 5: KSPLIT(6, 4, 3); break;
    case 6: KSPLIT(4, 4, 4); break;
    case 7: KSPLIT(4, 2, 6); break;
    case 8: KSPLIT(2, 4, 6); break;
    default: KSPLIT(2, 2, 6); break;
  }
#undef PINGPONG
#undef KSPLIT
  TB_LAUNCH_CHECK("linear_i8");
  if (part) {
    splitk_i8_kernel<<<(unsigned)cdiv(M * (Np / 8), 256), 256, 0, st>>>((const intx4*)part, p.splits, sx, ws, bi, yo, ldy, (int)M,
                                                                        (int)N, (int)Np);
    TB_LAUNCH_CHECK("linear_i8 split-K sum");
  }
  return 0;
}
