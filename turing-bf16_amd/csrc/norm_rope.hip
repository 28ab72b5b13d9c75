// RMS norm of every query and key head and rotation by position, in one pass, and its gradient.
//
// With x a head of D elements, w the weights, r = 1 / sqrt(mean x^2 + eps), u = x r:
//   z = u w,   y = z with its first R elements rotated: (y_i, y_j) = (z_i c - z_j s, z_j c + z_i s) for
//   pairs (i, j) = (p, p + R / 2), or neighbours (2 p, 2 p + 1), c and s row `position` of two tables.
// Gradient, dz being dy rotated back:
//   dw = sum over tokens and heads of dz u,   dx = r (dw' - u mean(dw' u)) with dw' = dz w.
//
// Bound by memory: 4 bytes an element forward, 6 backward, against ~8 and ~16 operations. A lane holds two
// chunks of 8 elements of a head, chosen so that a pair's elements are in one lane; L lanes
// make a head, whose sums go through DPP; a wave takes a token's heads, 64 / L at a time, so that
// cos and sin are read once for all of them and the weights once per wave.
// 8192 tokens of 40 heads of 128: 34.3 us, 5.0 TB/s; gradient of 8192 tokens of 32 heads: 41 us, 4.9 TB/s, and 4 us
// for the sums of the weights' (a copy reaches 4.9). 16 tokens: 5.9 us, the position, its angles and the store after
// one another.
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "abi_util.h"
#include "common.h"

using namespace tbf16;

namespace {

struct Heads {  // (B, S, heads, D) with element strides
  const uint16_t* x;
  int64_t sb, ss, sh;
};

struct NormArgs {
  Heads q, k, dyq, dyk;
  const void *wq, *wk;
  const float *cos, *sin;
  int64_t rows;  // of the tables
  const int32_t* pos;
  int64_t p_sb, p_ss;
  float eps, inv_d;
  int T, S, H, Hkv, D, R;
  int shares;  // forward: waves a token's steps go to
  uint16_t *yq, *yk;  // outputs, or dx of both
  int q_blocks;       // gradient: the first blocks take query heads, the others key heads
  float* part;        // [block][D], the blocks' shares of the weights' gradients
};

// Sum over the L lanes of a head, in each of them (DPP quad_perm, row_half_mirror, row_mirror).
template <int L>
__device__ __forceinline__ float sum_head(float v) {
  auto add = [&](auto ctrl) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xB1>());
  add(std::integral_constant<int, 0x4E>());
  if constexpr (L >= 8) add(std::integral_constant<int, 0x141>());
  if constexpr (L >= 16) add(std::integral_constant<int, 0x140>());
  return v;
}

// What a lane holds of a head: pairs (v[p], v[8 + p]) of chunks `lo` and `hi` of 8 elements.
template <bool NEAR>
struct Item {
  int lo, hi;   // elements
  bool there, turned;
  __device__ __forceinline__ Item(int i, int D, int R) {
    there = i < D / 16;
    turned = i < R / 16;
    lo = NEAR || !turned ? 16 * i : 8 * i;
    hi = NEAR || !turned ? 16 * i + 8 : 8 * i + R / 2;
  }
  // element of v[p]
  __device__ __forceinline__ int at(int p) const {
    if constexpr (NEAR) return ((p & 7) < 4 ? lo : hi) + 2 * (p & 3) + (p >> 3);
    return p < 8 ? lo + p : hi + p - 8;
  }
};
template <bool NEAR>
__device__ __forceinline__ void unpack(uint4 lo, uint4 hi, float* v) {
  const uint32_t d[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[NEAR ? i : 2 * i] = bf16_lo(d[i]);
    v[NEAR ? i + 8 : 2 * i + 1] = bf16_hi(d[i]);
  }
}
template <bool NEAR>
__device__ __forceinline__ void store(uint16_t* y, int lo, int hi, const float* v) {
  uint32_t d[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = NEAR ? pack_bf16(v[i], v[i + 8]) : pack_bf16(v[2 * i], v[2 * i + 1]);
  stg16(y + lo, make_uint4(d[0], d[1], d[2], d[3]));
  stg16(y + hi, make_uint4(d[4], d[5], d[6], d[7]));
}
template <bool NEAR, bool W32>
__device__ __forceinline__ void load_weights(const void* w, const Item<NEAR>& it, float* v) {
#pragma unroll
  for (int p = 0; p < 16; ++p) v[p] = 0.f;
  if (!it.there) return;
  if constexpr (W32) {
    float c[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + (i < 2 ? it.lo : it.hi - 8) + 4 * i);
      c[4 * i] = f.x; c[4 * i + 1] = f.y; c[4 * i + 2] = f.z; c[4 * i + 3] = f.w;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[NEAR ? i / 2 + 8 * (i & 1) : i] = c[i];
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(w);
    unpack<NEAR>(ldg16(h + it.lo), ldg16(h + it.hi), v);
  }
}

// x -> x r; returns r, and in `scale` a power of two so that x's gradient takes r scale. Squares that leave
// fp32's range (elements past 2^63, or below 2^-50 without an eps) are taken of x scaled by a power of two.
template <int L>
__device__ __forceinline__ float unit(float* x, float eps, float inv_d, float& scale) {
  auto mean = [&] {
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < 16; ++p) s = fmaf(x[p], x[p], s);
    return sum_head<L>(s) * inv_d;
  };
  float m = mean() + eps;
  scale = 1.f;
  if (__any(!(m >= 0x1p-100f && m <= FLT_MAX))) {
    scale = m >= 0x1p-100f && m <= FLT_MAX ? 1.f : m > 1.f ? 0x1p-80f : 0x1p80f;
#pragma unroll
    for (int p = 0; p < 16; ++p) x[p] *= scale;
    m = mean() + eps * scale * scale;
  }
  const float r = rsqrtf(m);
#pragma unroll
  for (int p = 0; p < 16; ++p) x[p] *= r;
  return r;
}

// A wave's place: the tables' row of a token.
struct Turn {
  float c[8], s[8];
};
template <bool NEAR>
__device__ __forceinline__ void load_turn(const NormArgs& a, const Item<NEAR>& it, int i, int pos, Turn& t) {
  const bool known = pos < a.rows;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    t.c[p] = known ? 1.f : __int_as_float(0x7fc00000);  // no angle: NaN
    t.s[p] = 0.f;
  }
  if (!known || !it.turned) return;
  const int64_t at = (int64_t)pos * (a.R / 2) + 8 * i;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 c = *reinterpret_cast<const float4*>(a.cos + at + 4 * h);
    const float4 s = *reinterpret_cast<const float4*>(a.sin + at + 4 * h);
    t.c[4 * h] = c.x; t.c[4 * h + 1] = c.y; t.c[4 * h + 2] = c.z; t.c[4 * h + 3] = c.w;
    t.s[4 * h] = s.x; t.s[4 * h + 1] = s.y; t.s[4 * h + 2] = s.z; t.s[4 * h + 3] = s.w;
  }
}

template <int L, bool NEAR, bool W32, bool BACK>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormArgs a) {
  constexpr int HPW = 64 / L, U = BACK ? 2 : 4;
  __shared__ float s_dw[BACK ? 4 : 1][BACK ? 16 * L : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane % L, hl = lane / L;
  const Item<NEAR> it(i, a.D, a.R);
  // Forward: query heads, then key heads, in steps of HPW. Gradient: one kind a block, whose registers then
  // hold one set of weights and of their gradients (189 -> 151 registers, three waves a SIMD instead of two: 56 -> 41
  // us for 8192 tokens of 32 heads).
  const int sq = (a.H + HPW - 1) / HPW, sk = (a.Hkv + HPW - 1) / HPW;
  const bool key_block = BACK && (int)blockIdx.x >= a.q_blocks;
  int begin = key_block ? sq : 0, steps = BACK && !key_block ? sq : sq + sk;
  float w[BACK ? 1 : 2][16], dw[16];
  load_weights<NEAR, W32>(key_block ? a.wk : a.wq, it, w[0]);
  if constexpr (BACK) {
#pragma unroll
    for (int p = 0; p < 16; ++p) dw[p] = 0.f;
  } else {
    load_weights<NEAR, W32>(a.wk, it, w[1]);
  }
  const int block = key_block ? blockIdx.x - a.q_blocks : blockIdx.x;
  const int blocks = !BACK ? gridDim.x : key_block ? gridDim.x - a.q_blocks : a.q_blocks;
  const int64_t tasks = BACK ? a.T : (int64_t)a.T * a.shares;
  for (int64_t tt = (int64_t)block * 4 + wave; tt < tasks; tt += (int64_t)blocks * 4) {
    int t = (int)tt;
    if (!BACK && a.shares > 1) {
      t = (int)(tt / a.shares);
      begin = (int)(tt - (int64_t)t * a.shares) * U;
      steps = min(begin + U, sq + sk);
    }
    const int b = t / a.S, s = t - b * a.S;
    const int pos_there = a.pos[b * a.p_sb + s * a.p_ss];
    int pos = 0;
    Turn turn;
    for (int st0 = begin; st0 < steps; st0 += U) {
      uint4 xv[U][2], gv[BACK ? U : 1][2];
      auto head_of = [&](int st) { return (st < sq ? st : st - sq) * HPW + hl; };
      auto valid = [&](int st) { return it.there && st < steps && head_of(st) < (st < sq ? a.H : a.Hkv); };
      if (st0 == begin || pos >= 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int st = st0 + u;
          xv[u][0] = xv[u][1] = make_uint4(0, 0, 0, 0);
          if constexpr (BACK) gv[u][0] = gv[u][1] = make_uint4(0, 0, 0, 0);
          if (!valid(st)) continue;
          const Heads& x = st < sq ? a.q : a.k;
          const uint16_t* at = x.x + b * x.sb + s * x.ss + head_of(st) * x.sh;
          xv[u][0] = ldg16(at + it.lo);
          xv[u][1] = ldg16(at + it.hi);
          if constexpr (BACK) {
            const Heads& g = st < sq ? a.dyq : a.dyk;
            const uint16_t* from = g.x + b * g.sb + s * g.ss + head_of(st) * g.sh;
            gv[u][0] = ldg16(from + it.lo);
            gv[u][1] = ldg16(from + it.hi);
          }
        }
      }
      if (st0 == begin) {  // (the first heads are on their way by now, whether or not the token is padding)
        pos = __builtin_amdgcn_readfirstlane(pos_there);
        if (pos >= 0) load_turn<NEAR>(a, it, i, pos, turn);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int st = st0 + u;
        if (st >= steps) break;
        const bool is_k = BACK ? key_block : st >= sq;
        const float* const ws = w[BACK ? 0 : is_k];
        uint16_t* out = is_k ? a.yk : a.yq;
        if (out) out += ((int64_t)t * (is_k ? a.Hkv : a.H) + head_of(st)) * a.D;
        float x[16];
        if (pos < 0) {  // padding
#pragma unroll
          for (int p = 0; p < 16; ++p) x[p] = 0.f;
          if (out && valid(st)) store<NEAR>(out, it.lo, it.hi, x);
          continue;
        }
        unpack<NEAR>(xv[u][0], xv[u][1], x);
        float scale;
        const float r = unit<L>(x, a.eps, a.inv_d, scale);
        if constexpr (!BACK) {
          float y[16];
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const float za = x[p] * ws[p], zb = x[8 + p] * ws[8 + p];
            y[p] = za * turn.c[p] - zb * turn.s[p];
            y[8 + p] = zb * turn.c[p] + za * turn.s[p];
          }
          if (valid(st)) store<NEAR>(out, it.lo, it.hi, y);
        } else {
          float g[16], d[16], dot = 0.f;
          unpack<NEAR>(gv[u][0], gv[u][1], g);
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            d[p] = g[p] * turn.c[p] + g[8 + p] * turn.s[p];
            d[8 + p] = g[8 + p] * turn.c[p] - g[p] * turn.s[p];
          }
          const bool mine = valid(st);  // (elsewhere x r may be NaN: zeros without an eps)
#pragma unroll
          for (int p = 0; p < 16; ++p) {
            dw[p] += mine ? d[p] * x[p] : 0.f;
            d[p] *= ws[p];
            dot = fmaf(d[p], x[p], dot);
          }
          dot = sum_head<L>(dot) * a.inv_d;
#pragma unroll
          for (int p = 0; p < 16; ++p) d[p] = (d[p] - x[p] * dot) * r * scale;
          if (out && mine) store<NEAR>(out, it.lo, it.hi, d);
        }
      }
    }
  }
  if constexpr (BACK) {
    if (a.part == nullptr) return;
#pragma unroll
    for (int p = 0; p < 16; ++p) {
      float v = dw[p];
#pragma unroll
      for (int o = L; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
      if (hl == 0 && it.there) s_dw[wave][it.at(p)] = v;
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d < a.D) a.part[(int64_t)blockIdx.x * a.D + d] = s_dw[0][d] + s_dw[1][d] + s_dw[2][d] + s_dw[3][d];
  }
}

// The blocks' shares of the weights' gradients, added in an order of their own: 16 columns of one kind a
// block, 64 threads each.
template <bool W32>
__global__ __launch_bounds__(1024) void norm_rope_weights_kernel(const float* part, int q_blocks, int blocks, int D, void* dwq,
                                                                 void* dwk) {
  __shared__ float s[64][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, d = blockIdx.x * 16 + c;
  const bool key = blockIdx.y;
  void* out = key ? dwk : dwq;
  if (out == nullptr) return;
  float v = 0.f;
#pragma unroll 4
  for (int b = (key ? q_blocks : 0) + g; b < (key ? blocks : q_blocks); b += 64) v += part[(int64_t)b * D + d];
  s[g][c] = v;
  __syncthreads();
  if (g == 0) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) v += s[i][c];
    if constexpr (W32) static_cast<float*>(out)[d] = v;
    else static_cast<uint16_t*>(out)[d] = (uint16_t)pack_bf16(v, 0.f);
  }
}

// As many as run at once, by the kinds' shares of the work.
struct BackBlocks {
  int64_t q, k;
};
BackBlocks backward_blocks(int64_t T, int64_t H, int64_t Hkv) {
  const int64_t all = 3 * num_cus(), most = cdiv(T, 4);
  const int64_t q = std::min(std::max<int64_t>(1, all * H / (H + Hkv)), all - 1);
  return {std::min(q, most), std::min(all - q, most)};
}

// Forward: blocks of four waves, a token a wave at a time; of few tokens each wave takes four steps' heads alone
// (16 tokens of 40 heads of 128: 6.4 -> 5.9 us).
int64_t forward_blocks(NormArgs& a) {
  const int heads = 64 / (a.D <= 64 ? 4 : a.D <= 128 ? 8 : 16), steps = (int)(cdiv(a.H, heads) + cdiv(a.Hkv, heads));
  a.shares = (int64_t)a.T * steps <= 16 * num_cus() ? (int)cdiv(steps, 4) : 1;
  return std::min<int64_t>(cdiv((int64_t)a.T * a.shares, 4), num_cus() * 8);
}

template <bool BACK>
void launch_norm(const NormArgs& a, int64_t blocks, bool near, bool w32, hipStream_t st) {
#define NORM(L_)                                                                       \
  do {                                                                                 \
    if (near && w32) norm_rope_kernel<L_, true, true, BACK><<<(unsigned)blocks, 256, 0, st>>>(a);   \
    else if (near) norm_rope_kernel<L_, true, false, BACK><<<(unsigned)blocks, 256, 0, st>>>(a);    \
    else if (w32) norm_rope_kernel<L_, false, true, BACK><<<(unsigned)blocks, 256, 0, st>>>(a);     \
    else norm_rope_kernel<L_, false, false, BACK><<<(unsigned)blocks, 256, 0, st>>>(a);             \
  } while (0)
  if (a.D <= 64) NORM(4);
  else if (a.D <= 128) NORM(8);
  else NORM(16);
#undef NORM
}

int check_norm(const char* fn, const NormArgs& a, int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int64_t R) {
  TB_CHECK(B >= 0 && S >= 0 && (double)B * (double)S < 2147483648.0, "%s: bad number of tokens", fn);
  TB_CHECK(H > 0 && Hkv > 0 && H < 1 << 20 && Hkv < 1 << 20, "%s: bad number of heads", fn);
  TB_CHECK(D > 0 && D <= 256 && D % 16 == 0, "%s: head dim must be a multiple of 16 up to 256", fn);
  TB_CHECK(R > 0 && R <= D && R % 16 == 0, "%s: rotated dims must be a multiple of 16 up to the head dim", fn);
  TB_CHECK(a.rows > 0, "%s: empty tables", fn);
  TB_CHECK(a.eps >= 0.f && a.eps <= FLT_MAX, "%s: bad eps", fn);
  for (const Heads* h : {&a.q, &a.k, &a.dyq, &a.dyk})
    TB_CHECK(aligned16(h->x) && h->sb % 8 == 0 && h->ss % 8 == 0 && h->sh % 8 == 0, "%s: rows must be 16-byte aligned", fn);
  TB_CHECK(aligned16(a.cos) && aligned16(a.sin) && aligned16(a.yq) && aligned16(a.yk) && aligned4(a.pos) && aligned16(a.wq) &&
               aligned16(a.wk) && aligned4(a.part),
           "%s: misaligned pointer", fn);
  return 0;
}

NormArgs norm_args(const Heads& q, const Heads& k, int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, const void* wq,
                   const void* wk, const float* cos, const float* sin, int64_t rows, int64_t R, const int32_t* pos,
                   int64_t p_sb, int64_t p_ss, float eps) {
  NormArgs a = {};
  a.q = q;
  a.k = k;
  a.wq = wq;
  a.wk = wk;
  a.cos = cos;
  a.sin = sin;
  a.rows = rows;
  a.pos = pos;
  a.p_sb = p_sb;
  a.p_ss = p_ss;
  a.eps = eps;
  a.inv_d = D > 0 ? 1.f / (float)D : 0.f;
  a.T = (int)(B * S);
  a.S = (int)S;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.D = (int)D;
  a.R = (int)R;
  return a;
}

}  // namespace

extern "C" int tbf16_qk_norm_rope(const void* q, const void* k, int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D,
                                  int64_t q_sb, int64_t q_ss, int64_t q_sh, int64_t k_sb, int64_t k_ss, int64_t k_sh,
                                  const void* wq, const void* wk, int w_f32, const float* cos, const float* sin,
                                  int64_t rows, int64_t R, const int32_t* pos, int64_t p_sb, int64_t p_ss, float eps,
                                  int interleaved, void* yq, void* yk, void* stream) {
  NormArgs a = norm_args({(const uint16_t*)q, q_sb, q_ss, q_sh}, {(const uint16_t*)k, k_sb, k_ss, k_sh}, B, S, H, Hkv, D, wq,
                         wk, cos, sin, rows, R, pos, p_sb, p_ss, eps);
  a.yq = (uint16_t*)yq;
  a.yk = (uint16_t*)yk;
  if (int rc = check_norm("qk_norm_rope", a, B, S, H, Hkv, D, R)) return rc;
  if (a.T == 0) return 0;
  const int64_t blocks = forward_blocks(a);
  launch_norm<false>(a, blocks, interleaved, w_f32, as_stream(stream));
  TB_LAUNCH_CHECK("qk_norm_rope");
  return 0;
}

extern "C" size_t tbf16_qk_norm_rope_bwd_ws_bytes(int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D) {
  if (B <= 0 || S <= 0 || H <= 0 || Hkv <= 0 || D <= 0 || (double)B * (double)S >= 2147483648.0) return 0;
  const BackBlocks n = backward_blocks(B * S, H, Hkv);
  return (size_t)(n.q + n.k) * (size_t)D * 4;
}

extern "C" int tbf16_qk_norm_rope_bwd(const void* q, const void* k, const void* dyq, const void* dyk, int64_t B, int64_t S,
                                      int64_t H, int64_t Hkv, int64_t D, int64_t q_sb, int64_t q_ss, int64_t q_sh,
                                      int64_t k_sb, int64_t k_ss, int64_t k_sh, int64_t dyq_sb, int64_t dyq_ss,
                                      int64_t dyq_sh, int64_t dyk_sb, int64_t dyk_ss, int64_t dyk_sh, const void* wq,
                                      const void* wk, int w_f32, const float* cos, const float* sin, int64_t rows, int64_t R,
                                      const int32_t* pos, int64_t p_sb, int64_t p_ss, float eps, int interleaved, void* dq,
                                      void* dk, void* dwq, void* dwk, void* ws, int64_t ws_bytes, void* stream) {
  NormArgs a = norm_args({(const uint16_t*)q, q_sb, q_ss, q_sh}, {(const uint16_t*)k, k_sb, k_ss, k_sh}, B, S, H, Hkv, D, wq,
                         wk, cos, sin, rows, R, pos, p_sb, p_ss, eps);
  a.dyq = {(const uint16_t*)dyq, dyq_sb, dyq_ss, dyq_sh};
  a.dyk = {(const uint16_t*)dyk, dyk_sb, dyk_ss, dyk_sh};
  a.yq = (uint16_t*)dq;
  a.yk = (uint16_t*)dk;
  const bool weights = dwq != nullptr || dwk != nullptr;
  a.part = weights ? (float*)ws : nullptr;
  if (int rc = check_norm("qk_norm_rope_bwd", a, B, S, H, Hkv, D, R)) return rc;
  TB_CHECK(aligned4(dwq) && aligned4(dwk), "qk_norm_rope_bwd: misaligned pointer");
  const BackBlocks n = a.T > 0 ? backward_blocks(a.T, H, Hkv) : BackBlocks{0, 0};
  const size_t need = tbf16_qk_norm_rope_bwd_ws_bytes(B, S, H, Hkv, D);
  if (weights && need && (ws == nullptr || ws_bytes < (int64_t)need)) {
    set_error("qk_norm_rope_bwd: workspace too small (%lld bytes, needs %zu)", (long long)ws_bytes, need);
    return TBF16_EWS;
  }
  a.q_blocks = (int)n.q;
  const hipStream_t st = as_stream(stream);
  if (a.T > 0) {
    launch_norm<true>(a, n.q + n.k, interleaved, w_f32, st);
    TB_LAUNCH_CHECK("qk_norm_rope_bwd");
  }
  if (weights) {  // (without tokens: zeros)
    const dim3 grid((unsigned)(D / 16), 2);
    const int blocks = (int)(n.q + n.k);
    if (w_f32) norm_rope_weights_kernel<true><<<grid, 1024, 0, st>>>(a.part, a.q_blocks, blocks, (int)D, dwq, dwk);
    else norm_rope_weights_kernel<false><<<grid, 1024, 0, st>>>(a.part, a.q_blocks, blocks, (int)D, dwq, dwk);
    TB_LAUNCH_CHECK("qk_norm_rope_bwd weights");
  }
  return 0;
}
