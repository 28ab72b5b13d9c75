// Tile kernels of the GEMMs on operands that need no conversion: c[m, n] = sum_k a[m, k] b[n, k],
// both operands K-contiguous, on fp16 (fp32 sums) or 8-bit integers (int32 sums). An operand row is
// counted in units of 2 bytes either way (K, row strides), a k tile is 128 bytes: 64 fp16 or 128
// integers, one MFMA of 64 bytes a row taking 32 or 64 of them. The two kinds share every tile,
// schedule and address, and differ in the MFMA, the sums' type and the factors of the epilogue.
#pragma once
#include <type_traits>

#include "common.h"

namespace tbf16 {

typedef int intx4 __attribute__((ext_vector_type(4)));

struct F16Op {
  typedef half8 Frag;
  typedef floatx4 Acc;
  static constexpr float kA = 1.f, kB = 1.f;
  static __device__ __forceinline__ Acc mma(Frag b, Frag a, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(b, a, c, 0, 0, 0);
  }
};
// kA, kB: the row factor times 2^-24 and the column factor times 2^24, so that a sum of up to
// 31 bits times a row's factor stays in fp32's range for every bf16 row.
struct I8Op {
  typedef intx4 Frag;
  typedef intx4 Acc;
  static constexpr float kA = 0x1p-24f, kB = 0x1p24f;
  static __device__ __forceinline__ Acc mma(Frag b, Frag a, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, c, 0, 0, 0);
  }
};

// Byte offset of 16-byte chunk `chunk` of row `row` in a [rows][BK] fp16 tile.
// BK = 64: 128-byte rows, chunk ^= (row / 2) % 8; BK = 32: 64-byte rows,
// chunk ^= (row / 4) % 4. Either way 16 lanes reading 16 consecutive rows at one
// logical chunk, or 8 (4) lanes writing one row, touch 64 distinct banks.
template <int BK>
__device__ __forceinline__ int swz(int row, int chunk) {
  if constexpr (BK == 64) return row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4);
  else return row * 64 + ((chunk ^ ((row >> 2) & 3)) << 4);
}

// Epilogue of a wave's TM x TN sub-tile made of 16x16 MFMA blocks: acc[i][j] holds
// columns 16 i and rows 16 j, lane l columns 4 (l / 16) .. + 3 of row l % 16. The same
// fp32 arithmetic as gemm.hip's store_tile; part: the raw sums, row stride ldp.
// v_permlane16_swap pairs column blocks 2 p and 2 p + 1 between 16-lane rows, so a lane holds 16 bytes of its row (columns 0 / 16 / 8 / 24 of
// the 32-column pair for l / 16 = 0 / 1 / 2 / 3); with two pairs, a DPP row_ror:8
// exchange between lanes l and l ^ 8 makes each store write whole 128-byte rows.
template <int TM, int TN, class V>
__device__ __forceinline__ void store_tile16(const V (&acc)[TN / 16][TM / 16], const float* sa_l, const float* sb_l,
                                             const uint16_t* bias_l, int wm, int wn, int lane, int m0, int n0,
                                             uint16_t* __restrict__ C, int64_t ldc, int M, int N, float* part, int ldp) {
  constexpr int FM = TM / 16, FN = TN / 16, NP = FN / 2;
  static_assert(FN == 2 || FN == 4, "sub-tile columns");
  const int fr = lane & 15, fk = lane >> 4;
  if (part) {
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int m = m0 + wm * TM + j * 16 + fr;
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int n = n0 + wn * TN + i * 16 + 4 * fk;
        if (m < M && n < N)
          *reinterpret_cast<V*>(part + (int64_t)m * ldp + n) = acc[i][j];
      }
    }
    return;
  }
  const int cl = ((fk & 1) << 4) | ((fk >> 1) << 3);
  const bool hi8 = (lane & 8) != 0;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const float sa = sa_l[wm * TM + j * 16 + fr];
    uint32_t v[NP][4];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      uint32_t w[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int nl = wn * TN + (2 * p + i) * 16 + 4 * fk;
        const float4 sb = *reinterpret_cast<const float4*>(sb_l + nl);
        const uint2 bw = *reinterpret_cast<const uint2*>(bias_l + nl);
        const V c = acc[2 * p + i][j];
        w[i][0] = pack_bf16(fmaf((float)c[0] * sa, sb.x, bf16_lo(bw.x)), fmaf((float)c[1] * sa, sb.y, bf16_hi(bw.x)));
        w[i][1] = pack_bf16(fmaf((float)c[2] * sa, sb.z, bf16_lo(bw.y)), fmaf((float)c[3] * sa, sb.w, bf16_hi(bw.y)));
      }
      const auto d0 = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
      const auto d1 = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
      v[p][0] = d0[0]; v[p][1] = d1[0]; v[p][2] = d0[1]; v[p][3] = d1[1];
    }
    const int row0 = m0 + wm * TM + j * 16, col0 = n0 + wn * TN + cl;
    if constexpr (NP == 2) {
      uint32_t f[4], g[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t t0 = __builtin_amdgcn_mov_dpp((int)v[0][d], 0x128, 0xF, 0xF, false);
        const uint32_t t1 = __builtin_amdgcn_mov_dpp((int)v[1][d], 0x128, 0xF, 0xF, false);
        f[d] = hi8 ? t1 : v[0][d];
        g[d] = hi8 ? v[1][d] : t0;
      }
      const int m = row0 + (lane & 7), n = col0 + (hi8 ? 32 : 0);
      if (n < N) {
        if (m < M) stg16(C + (int64_t)m * ldc + n, make_uint4(f[0], f[1], f[2], f[3]));
        if (m + 8 < M) stg16(C + (int64_t)(m + 8) * ldc + n, make_uint4(g[0], g[1], g[2], g[3]));
      }
    } else {
      if (row0 + fr < M && col0 < N)
        stg16(C + (int64_t)(row0 + fr) * ldc + col0, make_uint4(v[0][0], v[0][1], v[0][2], v[0][3]));
    }
  }
}

// Ping-pong GEMM (figures: fp16): 8 waves in two groups of four, one wave of each
// group per SIMD (waves w and w + 4 share a SIMD), half a phase apart: while one
// group's MFMAs run, the other reads its next fragments from LDS and issues direct
// global -> LDS loads; a bare barrier ends each such interval. Group g owns rows
// [BM / 2 g, + BM / 2) of the tile, wave w % 4 of it BN / 4 columns. k tile 64.
//  - MFMA 16x16x32: under this kernel the chip's clock is set by power, and the 16x16
//    form costs less of it than 32x32x16 (4096^3: 1.92 GHz and 101.8 us against 1.63
//    GHz and 113.4 us with the same schedule, same output bits).
//  - a k tile is staged as four half tiles, each its own __shared__ object: A half h
//    holds rows RA h .. + RA of each group's 2 RA, B half h columns CB h .. + CB of each
//    wave's 2 CB. S stages in a ring (tile kt in stage kt % S).
//  - a k tile is two phases, each one half of A against both of B (256x256: 32 MFMAs,
//    512 cycles). The B half 0 of a tile is read one phase early, which evens out
//    the LDS reads of the phases:
//      phase  MFMAs     reads                    loads
//      0      A0 B0 B1  A0, B1                   A1 of tile kt + S - 1, B0 of kt + S
//      1      A1 B0 B1  A1, B0 of tile kt + 1    A0, B1 of tile kt + S
//    A wave waits for its fragment reads (lgkmcnt 0) before the barrier that starts
//    its MFMAs; the other group's reads of the same phase are complete one barrier
//    later, so the next phase's loads may overwrite what this phase read.
//  - a half tile is loaded 2 S - 1 phases before it is read. Before each phase's first
//    barrier a wave waits until only the last 2 S - 2 phases' loads are left: what the
//    next phase reads has then landed for every wave of both groups. S = 2 is all
//    that fits at 256x256 and 192x256 (their phases are long enough to cover a load);
//    the smaller tiles' shorter phases need the deeper ring.
// Loads of tiles past the last go to a resource of length 0 (no memory traffic, zeros
// nobody reads). The fp32 additions run over k in ascending order.
// HA, FB: 16-row and 16-column blocks per wave and half (BM = 64 HA, BN = 128 FB).
// part / kt_per: split K, as gemm_kernel. NB <= N: rows of b, N rounded up to 8 (the
// columns past NB are zeros plus the last bias, for the caller to leave out).
template <class Op, int HA, int FB, int S, bool KEVEN>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void pingpong_kernel(
    const uint16_t* __restrict__ A, int64_t lda, const float* __restrict__ a_sinv, const uint16_t* __restrict__ B,
    int64_t ldb, const float* __restrict__ b_sinv, const uint16_t* __restrict__ bias, uint16_t* __restrict__ C,
    int64_t ldc, int M, int N, int K_all, float* __restrict__ part, int kt_per, int NB) {
  constexpr int BM = 64 * HA, BN = 128 * FB, RA = 16 * HA, CB = 16 * FB;
  constexpr int AB = 4 * HA, BB = 8 * FB;  // 1 KB blocks (8 rows of 128 bytes) of a half tile
  constexpr int AL = (AB + 7) / 8, BL = BB / 8;
  constexpr int INFLIGHT = (S - 1) * (HA + 2 * FB);  // a wave's loads of 2 S - 2 phases
  static_assert(HA >= 2 && HA <= 4 && (FB == 1 || FB == 2) && S >= 2 && S <= 4, "tile");
  __shared__ __align__(1024) uint8_t a00[AB * 1024], a01[AB * 1024], a10[AB * 1024], a11[AB * 1024];  // [stage][half]
  __shared__ __align__(1024) uint8_t b00[BB * 1024], b01[BB * 1024], b10[BB * 1024], b11[BB * 1024];
  constexpr int A2 = S > 2 ? AB * 1024 : 16, B2 = S > 2 ? BB * 1024 : 16, A3 = S > 3 ? AB * 1024 : 16,
                B3 = S > 3 ? BB * 1024 : 16;
  __shared__ __align__(1024) uint8_t a20[A2], a21[A2], a30[A3], a31[A3], b20[B2], b21[B2], b30[B3], b31[B3];
  uint8_t* const sa0[4] = {a00, a10, a20, a30};
  uint8_t* const sa1[4] = {a01, a11, a21, a31};
  uint8_t* const sb0[4] = {b00, b10, b20, b30};
  uint8_t* const sb1[4] = {b01, b11, b21, b31};
  __shared__ __align__(16) float sa_l[BM], sb_l[BN];
  __shared__ __align__(16) uint16_t bias_l[BN];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;  // wm: the group

  // tile assignment: XCD-contiguous ranges, then grouped raster (as gemm_kernel)
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (N + BN - 1) / BN;
  int bid = blockIdx.x;
  const int nblk = gridDim.x;
  if ((nblk & 7) == 0) bid = (bid & 7) * (nblk >> 3) + (bid >> 3);
  constexpr int GM = 8;
  const int group = bid / (GM * tiles_n), first = group * GM, gsize = min(tiles_m - first, GM);
  const int within = bid % (GM * tiles_n);
  const int m0 = (first + within % gsize) * BM;
  const int n0 = (within / gsize) * BN;
  const int ks = part ? (int)blockIdx.y : 0;
  const int kbase = ks * kt_per * 64;
  const int K = part ? min(K_all - kbase, kt_per * 64) : K_all;

  // the epilogue's factors, one a thread, loaded ahead of the direct loads (rows past M
  // and columns past N take the last one's and are not stored)
  const int fc = tid - 256;
  const float fsc = fc < 0 ? a_sinv[min(m0 + tid, M - 1)] * Op::kA : b_sinv[min(n0 + fc, NB - 1)] * Op::kB;
  const uint16_t fbias = bias ? bias[min(n0 + max(fc, 0), NB - 1)] : (uint16_t)0;

  // direct loads: lane l of the load of 1 KB block b lands at row 8 b + l / 8 of the
  // half tile, physical chunk l % 8, so it fetches the logical chunk `chunk` (the XOR
  // swizzle on the source side; a wave's blocks all have its own parity). Wave w loads
  // blocks w and w + 8; of 12 blocks (HA = 3) the last four are waves 0-3's in half 0
  // and waves 4-7's in half 1, so that every wave has the same loads in two phases.
  const int l8 = lane >> 3, chunk = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
  int aoff[2][AL], boff[2][BL];  // [half][block]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < AL; ++i) {
      const int r = 8 * (i == 0 ? wave : AB == 12 ? 8 + (wave & 3) : 8 + wave) + l8;
      aoff[h][i] = ((r / RA * 2 * RA + RA * h + r % RA) * (int)lda + chunk * 8) * 2;
    }
#pragma unroll
    for (int i = 0; i < BL; ++i) {
      const int r = 8 * (wave + 8 * i) + l8;
      boff[h][i] = ((r / CB * 2 * CB + CB * h + r % CB) * (int)ldb + chunk * 8) * 2;
    }
  }
  const BufRes ares =
      make_res(A + (int64_t)m0 * lda + kbase, min<int64_t>((int64_t)(M - m0) * lda * 2 - kbase * 2, 0x7fffffff));
  const BufRes bres =
      make_res(B + (int64_t)n0 * ldb + kbase, min<int64_t>((int64_t)(NB - n0) * ldb * 2 - kbase * 2, 0x7fffffff));
  const int KT = (K + 63) / 64;
  auto aload = [&](int h, uint8_t* half, int kt) {
    const BufRes rt{ares.lo, ares.hi, kt < KT ? ares.bytes : 0};
    const uint32_t base = lds_addr(half);
    const bool kok = KEVEN || kt * 64 + chunk * 8 < K;  // a k tail reads zeros
    buf_load16_lds(rt, base + wave * 1024, kok ? aoff[h][0] : (int)0x80000000, kt * 128);
    if constexpr (AB == 12) {
      if (wm == h) buf_load16_lds(rt, base + (8 + wn) * 1024, kok ? aoff[h][AL - 1] : (int)0x80000000, kt * 128);
    } else if constexpr (AB == 16) {
      buf_load16_lds(rt, base + (8 + wave) * 1024, kok ? aoff[h][AL - 1] : (int)0x80000000, kt * 128);
    }
  };
  auto bload = [&](int h, uint8_t* half, int kt) {
    const BufRes rt{bres.lo, bres.hi, kt < KT ? bres.bytes : 0};
    const uint32_t base = lds_addr(half);
    const bool kok = KEVEN || kt * 64 + chunk * 8 < K;
#pragma unroll
    for (int i = 0; i < BL; ++i)
      buf_load16_lds(rt, base + (wave + 8 * i) * 1024, kok ? boff[h][i] : (int)0x80000000, kt * 128);
  };

  typedef typename Op::Frag Frag;
  typename Op::Acc acc[2 * FB][2 * HA];  // [16 columns][16 rows]
#pragma unroll
  for (int i = 0; i < 2 * FB; ++i)
#pragma unroll
    for (int j = 0; j < 2 * HA; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = 0;

  const int fr = lane & 15, fk = lane >> 4;
  Frag fa[2][HA], fb0[2][2][FB], fb1[2][FB];  // [k step][block]; B0 of the current and the next tile
  auto areads = [&](const uint8_t* half) {
#pragma unroll
    for (int j = 0; j < HA; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        fa[s][j] = *reinterpret_cast<const Frag*>(half + swz<64>(wm * RA + j * 16 + fr, 4 * s + fk));
  };
  auto breads = [&](Frag(&f)[2][FB], const uint8_t* half) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < FB; ++i)
        f[s][i] = *reinterpret_cast<const Frag*>(half + swz<64>(wn * CB + i * 16 + fr, 4 * s + fk));
  };
  // a phase's MFMAs between its two barriers
  auto mma = [&](const Frag(&b0)[2][FB], int ha) {
    wait_vmem_n<INFLIGHT>();
    wait_lds();
    __builtin_amdgcn_sched_barrier(0);
    barrier_no_fence();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < HA; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 2 * FB; ++i)
          acc[i][HA * ha + j] = Op::mma(i < FB ? b0[s][i] : fb1[s][i - FB], fa[s][j], acc[i][HA * ha + j]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    barrier_no_fence();
    __builtin_amdgcn_sched_barrier(0);
  };

  // prologue: tiles 0 .. S - 2 whole, three half tiles of tile S - 1
#pragma unroll
  for (int t = 0; t < S; ++t) {
    bload(0, sb0[t], t);
    aload(0, sa0[t], t);
    bload(1, sb1[t], t);
    if (t + 1 < S) aload(1, sa1[t], t);
  }
  if (fc < 0) {
    if (tid < BM) sa_l[tid] = fsc;
  } else if (fc < BN) {
    sb_l[fc] = fsc;
    bias_l[fc] = fbias;
  }
  wait_vmem_n<INFLIGHT>();
  wait_lds();
  __builtin_amdgcn_sched_barrier(0);
  barrier_no_fence();
  __builtin_amdgcn_sched_barrier(0);
  breads(fb0[0], sb0[0]);
  wait_lds();
  __builtin_amdgcn_sched_barrier(0);
  barrier_no_fence();  // every wave has read B0 of tile 0: phase 0 loads over it
  if (wm == 1) barrier_no_fence();
  __builtin_amdgcn_sched_barrier(0);

  // tile kt in stage u % S; fb0[u % 2] holds its B0 fragments, fb0[(u + 1) % 2] takes tile kt + 1's
  constexpr int UN = S == 3 ? 6 : S;
  for (int kt0 = 0; kt0 < KT; kt0 += UN) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int kt = kt0 + u, c = u % S;
      if (u > 0 && kt >= KT) break;
      areads(sa0[c]);
      breads(fb1, sb1[c]);
      aload(1, sa1[(c + S - 1) % S], kt + S - 1);
      bload(0, sb0[c], kt + S);
      mma(fb0[u & 1], 0);
      areads(sa1[c]);
      breads(fb0[(u + 1) & 1], sb0[(c + 1) % S]);
      aload(0, sa0[c], kt + S);
      bload(1, sb1[c], kt + S);
      mma(fb0[u & 1], 1);
    }
  }
  if (wm == 0) barrier_no_fence();
  wait_vmem_n<0>();  // the loads of tiles past the last have ended before the block's LDS is given back
  store_tile16<2 * RA, 2 * CB>(acc, sa_l, sb_l, bias_l, wm, wn, lane, m0, n0, C, ldc, M, N,
                               part ? part + (int64_t)ks * M * N : nullptr, N);
}

// Where an implicit convolution's output pixels lie in its zero-padded channels-last
// input, in elements: `image` one image, row_step / col_step from one output row / column
// to the next; in bytes: next_col / next_row from the end of one tap's `chunks` 64-channel
// chunks (of one row's KW taps) to the start of the next.
struct ConvGeom {
  int64_t image = 0, out_image = 0;
  int Wo = 1, row_step = 0, col_step = 0, KW = 1, chunks = 1, next_col = 0, next_row = 0;
  const int32_t* exps = nullptr;
};

// store_tile16 for an implicit convolution: bf16(acc * sc[channel] + bias[channel]), channels
// along columns (CONV 1) or rows (CONV 2); rows of y at any alignment, the last columns
// one by one.
template <int TM, int TN, int CONV>
__device__ __forceinline__ void store_conv(const floatx4 (&acc)[TN / 16][TM / 16], const float* sc_l, const float* cb_l,
                                           int wm, int wn, int lane, int m0, int n0, uint16_t* __restrict__ C, int64_t ldc,
                                           int M, int N) {
  constexpr int FM = TM / 16, FN = TN / 16, NP = FN / 2;
  const int fr = lane & 15, fk = lane >> 4;
  const int cl = ((fk & 1) << 4) | ((fk >> 1) << 3);
  const bool hi8 = (lane & 8) != 0;
  auto put = [&](int m, int n, const uint32_t (&v)[4]) {
    if (m >= M || n >= N) return;
    uint16_t* const dst = C + (int64_t)m * ldc + n;
    if (n + 8 <= N) {
      __builtin_memcpy(dst, v, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < N) dst[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  };
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int ml = wm * TM + j * 16 + fr;
    uint32_t v[NP][4];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      uint32_t w[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const floatx4 c = acc[2 * p + i][j];
        float4 sc, cb;
        if constexpr (CONV == 1) {
          const int nl = wn * TN + (2 * p + i) * 16 + 4 * fk;
          sc = *reinterpret_cast<const float4*>(sc_l + nl);
          cb = *reinterpret_cast<const float4*>(cb_l + nl);
        } else {
          sc.x = sc.y = sc.z = sc.w = sc_l[ml];
          cb.x = cb.y = cb.z = cb.w = cb_l[ml];
        }
        w[i][0] = pack_bf16(fmaf(c[0], sc.x, cb.x), fmaf(c[1], sc.y, cb.y));
        w[i][1] = pack_bf16(fmaf(c[2], sc.z, cb.z), fmaf(c[3], sc.w, cb.w));
      }
      const auto d0 = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
      const auto d1 = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
      v[p][0] = d0[0]; v[p][1] = d1[0]; v[p][2] = d0[1]; v[p][3] = d1[1];
    }
    const int row0 = m0 + wm * TM + j * 16, col0 = n0 + wn * TN + cl;
    if constexpr (NP == 2) {
      uint32_t f[4], g[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t t0 = __builtin_amdgcn_mov_dpp((int)v[0][d], 0x128, 0xF, 0xF, false);
        const uint32_t t1 = __builtin_amdgcn_mov_dpp((int)v[1][d], 0x128, 0xF, 0xF, false);
        f[d] = hi8 ? t1 : v[0][d];
        g[d] = hi8 ? v[1][d] : t0;
      }
      const int n = col0 + (hi8 ? 32 : 0);
      put(row0 + (lane & 7), n, f);
      put(row0 + (lane & 7) + 8, n, g);
    } else {
      put(row0 + fr, col0, v[0]);
    }
  }
}

// Ping-pong GEMM for tiles too small for pingpong_kernel's phases:
// both groups of four waves (2 x 2 sub-tiles of 16 RM x 16 RN) cover the whole BM x BN
// tile, group 0 with the even k tiles, group 1 with the odd ones, and their sums meet
// in LDS at the end. Interval t (between two bare barriers): group t % 2 reads its
// fragments of tile t while the other group multiplies tile t - 1; every wave issues
// its share of the direct loads of tile t + S - 1 into the stage of tile t - 1, whose
// reads ended before the interval began, and before the interval's barrier waits until
// tile t + 1 has landed (the loads of S - 2 later tiles are left in flight).
//  - a wave's sub-tile is twice as wide as with eight waves side by side: a third
//    less LDS traffic per product, and an interval holds a whole k tile of one group
//    (128x128: 32 MFMAs, 512 cycles) instead of a quarter.
//  - an odd number of k tiles is padded with one of zeros (a resource of length 0).
// The two groups' fp32 sums are added even + odd: another order than k ascending,
// the same for every launch. part / kt_per: split K, as gemm_kernel. R <= BN: columns
// per block (a multiple of 8); below BN the weights of a single row of tiles are
// spread over every CU, the rest of the tile is zeros. NB: as pingpong_kernel.
// CONV: an implicit convolution. 1: a's rows are output pixels (y is pixels x channels), 2:
// b's are (y is channels x pixels), one image per blockIdx.y; the other operand is the
// weight [channel][tap][Cp]. A pixel's k tile is 64 channels of one tap of the zero-
// padded channels-last input, so a row's loads start at its own top left element and
// every k tile adds the same offset to all of them (ConvGeom). The factors are 2^e[image]
// ws[channel] and the bias fp32.
template <class Op, int RM, int RN, int S, bool KEVEN, int CONV = 0>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void ksplit_kernel(
    const uint16_t* __restrict__ A, int64_t lda, const float* __restrict__ a_sinv, const uint16_t* __restrict__ B,
    int64_t ldb, const float* __restrict__ b_sinv, const uint16_t* __restrict__ bias, uint16_t* __restrict__ C,
    int64_t ldc, int M, int N_all, int K_all, float* __restrict__ part, int kt_per, int R, int NB, ConvGeom cg) {
  constexpr int BM = 32 * RM, BN = 32 * RN, TM = 16 * RM, TN = 16 * RN;
  constexpr int STG = (BM + BN) * 128, NL = (BM + BN) / 64, AL = BM / 64;  // loads per wave and tile; the first AL are A's
  constexpr int XB = RM / 2 * RN * 16 * 64;  // bytes of the half sub-tile a wave hands over
  static_assert(RM % 2 == 0 && (RN == 2 || RN == 4) && S >= 3 && S <= 9 && 3 * (STG / XB) >= 8 && NL * 64 == BM + BN, "tile");
  __shared__ __align__(1024) uint8_t st0[STG], st1[STG], st2[STG];
  __shared__ __align__(1024) uint8_t st3[S > 3 ? STG : 16], st4[S > 4 ? STG : 16], st5[S > 5 ? STG : 16];
  __shared__ __align__(1024) uint8_t st6[S > 6 ? STG : 16], st7[S > 7 ? STG : 16], st8[S > 8 ? STG : 16];
  __shared__ __align__(16) float sa_l[BM], sb_l[BN];
  __shared__ __align__(16) uint16_t bias_l[CONV ? 8 : BN];
  __shared__ __align__(16) float cbias_l[CONV == 1 ? BN : CONV == 2 ? BM : 4];
  uint8_t* const stages[9] = {st0, st1, st2, st3, st4, st5, st6, st7, st8};

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave >> 1) & 1, wn = wave & 1;

  // tile assignment: XCD-contiguous ranges, then grouped raster (as gemm_kernel)
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (N_all + R - 1) / R;
  int bid = blockIdx.x;
  const int nblk = gridDim.x;
  if ((nblk & 7) == 0) bid = (bid & 7) * (nblk >> 3) + (bid >> 3);
  constexpr int GM = 8;
  const int group = bid / (GM * tiles_n), first = group * GM, gsize = min(tiles_m - first, GM);
  const int within = bid % (GM * tiles_n);
  const int m0 = (first + within % gsize) * BM;
  const int n0 = (within / gsize) * R, N = min(N_all, n0 + R);
  const int ks = !CONV && part ? (int)blockIdx.y : 0;
  if constexpr (CONV == 1) A += (int64_t)blockIdx.y * cg.image;
  if constexpr (CONV == 2) B += (int64_t)blockIdx.y * cg.image;
  if constexpr (CONV != 0) C += (int64_t)blockIdx.y * cg.out_image;
  const int kbase = ks * kt_per * 64;
  const int K = part ? min(K_all - kbase, kt_per * 64) : K_all;

  // the epilogue's factors (see pingpong_kernel)
  const int fc = tid - 256;
  float fsc, fcb = 0.f;
  uint16_t fbias = 0;
  if constexpr (CONV != 0) {
    const int o = CONV == 1 ? min(n0 + (tid & 255), N_all - 1) : min(m0 + (tid & 255), M - 1);
    fsc = ldexp1(cg.exps[blockIdx.y]) * (CONV == 1 ? b_sinv : a_sinv)[o];
    if (bias) fcb = bf16_lo(bias[o]);
  } else {
    fsc = fc < 0 ? a_sinv[min(m0 + tid, M - 1)] * Op::kA : b_sinv[min(n0 + fc, NB - 1)] * Op::kB;
    if (bias) fbias = bias[min(n0 + max(fc, 0), NB - 1)];
  }

  // direct loads: 1 KB block wave + 8 i of the stage (rows of A, then of B)
  const int chunk = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
  int off[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = 8 * (wave + 8 * (i < AL ? i : i - AL)) + (lane >> 3);
    if ((CONV == 1 && i < AL) || (CONV == 2 && i >= AL)) {  // pixels past the last take the last's
      const int px = CONV == 1 ? min(m0 + r, M - 1) : min(n0 + r, N_all - 1);
      off[i] = (px / cg.Wo * cg.row_step + px % cg.Wo * cg.col_step + chunk * 8) * 2;
    } else {
      off[i] = (r * (int)(i < AL ? lda : ldb) + chunk * 8) * 2;
    }
  }
  const BufRes ares =
      CONV == 1 ? make_res(A, cg.image * 2)
                : make_res(A + (int64_t)m0 * lda + kbase, min<int64_t>((int64_t)(M - m0) * lda * 2 - kbase * 2, 0x7fffffff));
  const BufRes bres =
      CONV == 2 ? make_res(B, cg.image * 2)
                : make_res(B + (int64_t)n0 * ldb + kbase,
                           min<int64_t>((int64_t)(min(N, NB) - n0) * ldb * 2 - kbase * 2, 0x7fffffff));
  // byte offset of a pixel's k tile from its top left element; load() is called for the
  // k tiles in order by every wave
  int p_off = 0, p_chunk = 0, p_col = 0;
  const int KT = (K + 63) / 64;
  auto load = [&](uint8_t* stage, int kt) {
    const BufRes ra{ares.lo, ares.hi, kt < KT ? ares.bytes : 0}, rb{bres.lo, bres.hi, kt < KT ? bres.bytes : 0};
    const uint32_t base = lds_addr(stage) + wave * 1024;
    const bool kok = KEVEN || kt * 64 + chunk * 8 < K;  // a k tail reads zeros
#pragma unroll
    for (int i = 0; i < NL; ++i)
      buf_load16_lds(i < AL ? ra : rb, base + i * 8192, kok ? off[i] : (int)0x80000000,
                     (CONV == 1 && i < AL) || (CONV == 2 && i >= AL) ? p_off : kt * 128);
    if constexpr (CONV != 0) {
      p_off += 128;
      if (++p_chunk == cg.chunks) {
        p_chunk = 0;
        p_off += cg.next_col;
        if (++p_col == cg.KW) {
          p_col = 0;
          p_off += cg.next_row;
        }
      }
    }
  };

  typedef typename Op::Frag Frag;
  typedef typename Op::Acc Acc;
  Acc acc[RN][RM];  // [16 columns][16 rows]
#pragma unroll
  for (int i = 0; i < RN; ++i)
#pragma unroll
    for (int j = 0; j < RM; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = 0;
  const int fr = lane & 15, fk = lane >> 4;
  Frag fa[2][RM], fb[2][RN];
  auto settle = [&]() {  // the end of an interval
    wait_vmem_n<NL*(S - 2)>();
    wait_lds();
    __builtin_amdgcn_sched_barrier(0);
    barrier_no_fence();
    __builtin_amdgcn_sched_barrier(0);
  };

#pragma unroll
  for (int t = 0; t < S - 1; ++t) load(stages[t], t);
  if constexpr (CONV != 0) {
    if (tid < (CONV == 1 ? BN : BM)) {
      (CONV == 1 ? sb_l : sa_l)[tid] = fsc;
      cbias_l[tid] = fcb;
    }
  } else if (fc < 0) {
    if (tid < BM) sa_l[tid] = fsc;
  } else if (fc < BN) {
    sb_l[fc] = fsc;
    bias_l[fc] = fbias;
  }
  settle();

  const int J = (KT + 1) / 2;  // k tiles per group
  auto run = [&](auto g_c) {
    constexpr int g = decltype(g_c)::value;
    if constexpr (g == 1) {
      load(stages[S - 1], S - 1);
      settle();
    }
    constexpr int UN = S % 2 ? S : S / 2;
    for (int j0 = 0; j0 < J; j0 += UN) {
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        if (u > 0 && j0 + u >= J) break;
        const int kt = 2 * (j0 + u) + g;
        const int c = (2 * u + g) % S;
        const uint8_t* stage = stages[c];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int i = 0; i < RN; ++i)
            fb[s][i] = *reinterpret_cast<const Frag*>(stage + swz<64>(BM + wn * TN + i * 16 + fr, 4 * s + fk));
#pragma unroll
          for (int j = 0; j < RM; ++j)
            fa[s][j] = *reinterpret_cast<const Frag*>(stage + swz<64>(wm * TM + j * 16 + fr, 4 * s + fk));
        }
        load(stages[(c + S - 1) % S], kt + S - 1);
        settle();
        load(stages[c], kt + S);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < RM; ++j)
#pragma unroll
            for (int i = 0; i < RN; ++i)
              acc[i][j] = Op::mma(fb[s][i], fa[s][j], acc[i][j]);
        __builtin_amdgcn_s_setprio(0);
        settle();
      }
    }
    if constexpr (g == 0) settle();
    // hand the other group half of the rows' sums, take its sums of the rest
    wait_vmem_n<0>();
    __syncthreads();
    constexpr int H = RM / 2;
    constexpr int PER = STG / XB;  // waves' regions per stage
    auto region = [&](int w) {
      return reinterpret_cast<Acc*>((w < PER ? st0 : w < 2 * PER ? st1 : st2) + (w % PER) * XB) + lane;
    };
    Acc* const out = region(wave);
    const Acc* const in = region(wave ^ 4);
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
      for (int j = 0; j < H; ++j) out[(i * H + j) * 64] = acc[i][g ? j : H + j];
    __syncthreads();
    Acc sum[RN][H];
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const Acc v = in[(i * H + j) * 64], o = acc[i][g ? H + j : j];
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[i][j][r] = o[r] + v[r];  // even + odd (commutative: the same bits in either group)
      }
    // rows wm TM + g TM / 2 of the tile: sub-tile row 2 wm + g of height TM / 2
    if constexpr (CONV != 0)
      store_conv<TM / 2, TN, CONV>(sum, CONV == 1 ? sb_l : sa_l, cbias_l, 2 * wm + g, wn, lane, m0, n0, C, ldc, M, N);
    else
      store_tile16<TM / 2, TN>(sum, sa_l, sb_l, bias_l, 2 * wm + g, wn, lane, m0, n0, C, ldc, M, N,
                               part ? part + (int64_t)ks * M * N_all : nullptr, N_all);
  };
  if (wave < 4) run(std::integral_constant<int, 0>{});
  else run(std::integral_constant<int, 1>{});
}


}  // namespace tbf16
