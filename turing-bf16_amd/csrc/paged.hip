// A paged key/value cache: writing new tokens into it, and attention of one new token per
// sequence over it (paged_attn.h).
#include "paged_attn.h"

using namespace tbf16;

namespace {

// ---- write ------------------------------------------------------------------------

// A copy, bound by memory (8192 tokens of 8 heads of 128: 18.5 us, 3.6 TB/s, from HBM; 13.5 us where the rows
// are still in the on-chip cache). A block takes TB tokens: a
// thread one 16-byte chunk of the keys' or values' heads, over the block's tokens (W threads a token,
// so 256 / W tokens at once).
// A slot that a later token names too is left to that token, so a repeated slot holds the last one's
// whole rows whatever the order of the blocks: the block marks its slots in a table of bits (by their low
// 16 bits; with 11 the false hits cost more than the copy) and looks up every later token's slot
// there, those that hit it in full. That search grows with the square of the tokens, so more than
// kWriteTokens are written by launches in turn (84140 short rows: 72 us; by 16384 at once 90, floor 26).
constexpr int kWriteBlock = 32, kWriteTokens = 65536, kNamed = 65536;
__global__ __launch_bounds__(256) void paged_write_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                          int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                                                          const int32_t* __restrict__ slots, int T, int TB, int C, int D8,
                                                          int W, uint16_t* __restrict__ kc, uint16_t* __restrict__ vc,
                                                          CacheGeom kg, CacheGeom vg, int n_slots, int page) {
  __shared__ int mine[kWriteBlock];  // the block's slots, -1: nowhere
  __shared__ int64_t koff[kWriteBlock], voff[kWriteBlock];
  __shared__ uint32_t named[kNamed / 32];
  const int tid = threadIdx.x, t0 = blockIdx.x * TB, nt = min(TB, T - t0);
  for (int i = tid; i < kNamed / 32; i += 256) named[i] = 0;
  int slot = -1;
  if (tid < nt) {
    slot = slots[t0 + tid];
    if (slot >= n_slots) slot = -1;
    const int p = slot / page, r = slot % page;
    mine[tid] = slot;
    koff[tid] = p * kg.sp + r * kg.ss;
    voff[tid] = p * vg.sp + r * vg.ss;
  }
  __syncthreads();
  if (slot >= 0) atomicOr(&named[(slot % kNamed) >> 5], 1u << (slot & 31));
  __syncthreads();
  constexpr int U = 4;
  auto look = [&](int s, int u) {  // (threads that find the same loss write the same)
    if (s >= 0 && (named[(s % kNamed) >> 5] >> (s & 31) & 1))
      for (int t = 0; t < nt; ++t)
        if (mine[t] == s && t0 + t < u) mine[t] = -1;
  };
  int u0 = t0 + 1 + 4 * tid;
  for (; u0 - 4 * tid + 256 * 4 * U <= T; u0 += 256 * 4 * U) {
    int4 s[U];
#pragma unroll
    for (int i = 0; i < U; ++i) __builtin_memcpy(&s[i], slots + u0 + 1024 * i, 16);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = u0 + 1024 * i;
      look(s[i].x, u);
      look(s[i].y, u + 1);
      look(s[i].z, u + 2);
      look(s[i].w, u + 3);
    }
  }
  for (int u = u0 - 3 * tid; u < T; u += 256 * U) {
    int s[U];
#pragma unroll
    for (int i = 0; i < U; ++i) s[i] = u + 256 * i < T ? slots[u + 256 * i] : -1;
#pragma unroll
    for (int i = 0; i < U; ++i) look(s[i], u + 256 * i);
  }
  __syncthreads();
  for (int j = tid & (W - 1); j < 2 * C; j += W) {
    const bool is_v = j >= C;
    const int e = is_v ? j - C : j, h = e / D8, c = (e - h * D8) * 8;
    const uint16_t* src = (is_v ? v + t0 * v_st + h * v_sh : k + t0 * k_st + h * k_sh) + c;
    uint16_t* dst = (is_v ? vc + h * vg.sh : kc + h * kg.sh) + c;
    const int64_t st = is_v ? v_st : k_st;
    const int64_t* off = is_v ? voff : koff;
    const int step = 256 / W;
    for (int t = tid / W; t < nt; t += U * step) {
      uint4 x[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (t + i * step < nt && mine[t + i * step] >= 0) x[i] = ldg16(src + (t + i * step) * st);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (t + i * step < nt && mine[t + i * step] >= 0) stg16(dst + off[t + i * step], x[i]);
    }
  }
}

// ---- attention ----------------------------------------------------------------------

template <int DP, int RT, int WPB, bool PAD, bool UNIT>
__global__ __launch_bounds__(WPB * 64, DP == 256 ? 1 : DP == 64 && RT == 1 ? 4 : 2) void paged_attn_kernel(AttnArgs a) {
  extern __shared__ __align__(16) float lds[];
  __shared__ int flags[WPB];
  attn_block<DP, RT, WPB, PAD, UNIT, false>(
      a, [&](int w) { return lds + w * a.R * (DP + 4); }, lds + WPB * a.R * (DP + 4), flags, blockIdx.x, gridDim.x, blockIdx.y,
      blockIdx.z);
}

// The join between blocks: for the unit that block blockIdx.x of the list began and did not end,
// 64 groups of 4 outputs a block; its waves take the parts in turns and meet in LDS.
constexpr int kJoinWaves = 8;
__global__ __launch_bounds__(kJoinWaves * 64) void paged_join_kernel(AttnArgs a) {
  __shared__ float4 so[kJoinWaves][64];
  __shared__ float2 ss[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int4 u = a.desc[blockIdx.x];
  if (u.w == 0) return;
  const int first = blockIdx.x, last = min(u.z, (int)gridDim.x - 1), rows = unit_rows(a, u.w - 1), dg = a.D / 4;
  const int e = blockIdx.y * 64 + lane;  // (row, group of 4)
  const int row = min(e / dg, rows - 1), d = e % dg * 4;
  float m = kNone, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 s, float4 v) {
    const float mn = fmaxf(m, s.x), f = ex2(m - mn), h = ex2(s.x - mn);
    m = mn;
    l = fmaf(l, f, s.y * h);
    o.x = fmaf(o.x, f, v.x * h);
    o.y = fmaf(o.y, f, v.y * h);
    o.z = fmaf(o.z, f, v.z * h);
    o.w = fmaf(o.w, f, v.w * h);
  };
  constexpr int U = 4;  // parts in flight
  for (int i0 = first + wave; i0 <= last; i0 += U * kJoinWaves) {
    float2 s[U];
    float4 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = min(i0 + k * kJoinWaves, last);
      const int64_t slot = (int64_t)i * 2 + (i == first ? 1 : 0);
      s[k] = *reinterpret_cast<const float2*>(a.stat + (slot * a.R + row) * 2);
      v[k] = *reinterpret_cast<const float4*>(a.part + (slot * a.R + row) * a.D + d);
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (i0 + k * kJoinWaves <= last) add(s[k], v[k]);
  }
  so[wave][lane] = o;
  ss[wave][lane] = make_float2(m, l);
  __syncthreads();
  if (wave != 0 || e >= rows * dg) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) add(ss[w][lane], so[w][lane]);
  const float f = m == kNone ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(unit_out(a, u.x, u.y, u.w - 1) + (int64_t)row * a.D + d) =
      make_uint2(pack_bf16(o.x * f, o.y * f), pack_bf16(o.z * f, o.w * f));
}

AttnPlan attn_plan(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t cap) {
  AttnPlan p;
  const int64_t G = H / Hkv;
  p.DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  p.RT = G <= 16 || p.DP == 256 ? 1 : G <= 32 || p.DP == 128 ? 2 : 4;
  p.R = (int)std::min<int64_t>(G, 16 * p.RT);
  p.RG = (int)cdiv(G, p.R);
  p.wpb = p.DP == 256 || p.RT > 1 ? 4 : 8;
  // Few short units: a launch less on the host and on the device (1 x 32 heads, 100 keys: 5.5 us, the
  // list and its join 8.4); with more tiles a wave the list's finer split wins (700 keys of 16 heads, 3
  // tiles a wave: 12.6 and 9.9 us on the device, 12.6 and 16.1 with the host; at 1000 keys, 4 tiles, by 2.3)
  p.unit = cdiv(cap, kTile) <= 3 * p.wpb && B * Hkv * p.RG <= num_cus();
  p.stat = p.desc = p.bytes = 0;
  p.blocks = 0;
  if (p.unit) return p;
  // as many as run at once: by registers, 4 waves a SIMD of D = 64, 2 of D = 128, 1 of D = 256
  p.blocks = num_cus() * (p.DP == 64 || (p.wpb == 4 && p.DP < 256) ? 2 : 1);
  p.stat = align_up((size_t)p.blocks * 2 * p.R * (size_t)D * 4, 256);
  p.desc = p.stat + align_up((size_t)p.blocks * 2 * p.R * 2 * 4, 256);
  p.bytes = p.desc + align_up((size_t)p.blocks * 16, 256);
  return p;
}

template <int DP, int RT, int WPB>
void launch_rows(const AttnArgs& a, bool unit, int64_t blocks, hipStream_t st) {
  const dim3 grid = unit ? dim3((unsigned)a.B, (unsigned)a.Hkv, (unsigned)a.RG) : dim3((unsigned)blocks);
  const size_t lds = (size_t)WPB * a.R * (DP + 4 + 2) * 4;
  const bool pad = a.D != DP;
#define ATTN(PAD_, UNIT_) \
  paged_attn_kernel<DP, RT, WPB, PAD_, UNIT_><<<grid, WPB * 64, lds, st>>>(a)
  if (unit) {
    if (pad) ATTN(true, true);
    else ATTN(false, true);
  } else {
    if (pad) ATTN(true, false);
    else ATTN(false, false);
  }
#undef ATTN
}

void launch_attn(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
#define ATTN(DP_, RT_, WPB_) launch_rows<DP_, RT_, WPB_>(a, p.unit, p.blocks, st)
  if (p.DP == 64) {
    if (p.RT == 1) ATTN(64, 1, 8);
    else if (p.RT == 2) ATTN(64, 2, 4);
    else ATTN(64, 4, 4);
  } else if (p.DP == 128) {
    if (p.RT == 1) ATTN(128, 1, 8);
    else ATTN(128, 2, 4);
  } else {
    ATTN(256, 1, 4);
  }
#undef ATTN
}

}  // namespace

extern "C" int tbf16_paged_write(const void* k, const void* v, int64_t T, int64_t Hkv, int64_t D, int64_t k_st,
                                 int64_t k_sh, int64_t v_st, int64_t v_sh, const int32_t* slots, void* k_cache,
                                 void* v_cache, int64_t pages, int64_t page, int64_t kc_sp, int64_t kc_sh, int64_t kc_ss,
                                 int64_t vc_sp, int64_t vc_sh, int64_t vc_ss, void* stream) {
  const CacheGeom kg{kc_sp, kc_sh, kc_ss}, vg{vc_sp, vc_sh, vc_ss};
  if (int rc = check_cache("paged_write", k_cache, v_cache, pages, Hkv, page, D, kg, vg)) return rc;
  TB_CHECK(T >= 0 && T < (int64_t)1 << 31, "paged_write: bad number of tokens");
  TB_CHECK(aligned16(k) && aligned16(v) && aligned4(slots), "paged_write: k and v must be 16-byte aligned");
  TB_CHECK(k_st % 8 == 0 && k_sh % 8 == 0 && v_st % 8 == 0 && v_sh % 8 == 0, "paged_write: strides must be multiples of 8");
  TB_CHECK(pages * page < (int64_t)1 << 31, "paged_write: more slots than int32 counts");
  if (T == 0 || pages == 0) return 0;
  const int C = (int)(Hkv * (D / 8));
  int W = 1;
  while (W < 256 && W < 2 * C) W *= 2;
  for (int64_t t = 0; t < T; t += kWriteTokens) {
    const int n = (int)std::min<int64_t>(kWriteTokens, T - t);
    // 8 blocks a CU as long as there are tokens (16384 of 8 heads: 34.8 us; 4 blocks 38.5, 16 blocks 41.2)
    const int TB = (int)std::min<int64_t>(kWriteBlock, std::max<int64_t>(256 / W, n / (8 * num_cus())));
    paged_write_kernel<<<(unsigned)cdiv(n, TB), 256, 0, as_stream(stream)>>>(
        (const uint16_t*)k + t * k_st, (const uint16_t*)v + t * v_st, k_st, k_sh, v_st, v_sh, slots + t, n, TB, C, (int)(D / 8),
        W, (uint16_t*)k_cache, (uint16_t*)v_cache, kg, vg, (int)(pages * page), (int)page);
    TB_LAUNCH_CHECK("paged_write");
  }
  return 0;
}

extern "C" size_t tbf16_paged_attn_ws_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t positions) {
  return B > 0 && H > 0 && Hkv > 0 && D > 0 && H % Hkv == 0 ? attn_plan(B, H, Hkv, D, positions).bytes : 0;
}

extern "C" int tbf16_paged_attn(const void* q, int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t q_sb, int64_t q_sh,
                                const void* k_cache, const void* v_cache, int64_t pages, int64_t page, int64_t kc_sp,
                                int64_t kc_sh, int64_t kc_ss, int64_t vc_sp, int64_t vc_sh, int64_t vc_ss,
                                const int32_t* table, int64_t table_stride, int64_t max_pages, const int32_t* lengths,
                                float scale, void* o, void* ws, int64_t ws_bytes, void* stream) {
  const CacheGeom kg{kc_sp, kc_sh, kc_ss}, vg{vc_sp, vc_sh, vc_ss};
  TB_CHECK(B >= 0 && H > 0 && H < (int64_t)1 << 24, "paged_attn: bad shape");
  if (int rc = check_cache("paged_attn", k_cache, v_cache, pages, Hkv, page, D, kg, vg)) return rc;
  TB_CHECK(H % Hkv == 0, "paged_attn: query heads must be a multiple of key/value heads");
  TB_CHECK(D <= 256, "paged_attn: head dim must be at most 256");
  TB_CHECK(max_pages >= 0 && max_pages < (int64_t)1 << 31, "paged_attn: table too wide");
  TB_CHECK(aligned16(q) && aligned16(o) && q_sb % 8 == 0 && q_sh % 8 == 0,
           "paged_attn: q must have 16-byte aligned rows");
  TB_CHECK(aligned4(table) && aligned4(lengths), "paged_attn: table and lengths must be 4-byte aligned");
  if (B == 0) return 0;
  const AttnPlan p = attn_plan(B, H, Hkv, D, max_pages * page);
  TB_CHECK(aligned16(ws) && (ws != nullptr || p.bytes == 0), "paged_attn: workspace missing or misaligned");
  TB_CHECK(B < (int64_t)1 << 31 && B * Hkv * p.RG < (int64_t)1 << 31 &&
               (double)(B * Hkv * p.RG) * (double)cdiv(std::min<int64_t>(max_pages * page, (int64_t)1 << 31), kTile) < 2e9,
           "paged_attn: shape too large");
  if (ws_bytes < (int64_t)p.bytes) {
    set_error("paged_attn: workspace too small (%lld bytes, needs %zu)", (long long)ws_bytes, p.bytes);
    return TBF16_EWS;
  }
  const AttnArgs a = attn_args(p, q, B, H, Hkv, D, q_sb, q_sh, k_cache, v_cache, pages, page, kg, vg, table, table_stride,
                               max_pages, lengths, scale, o, ws);
  const hipStream_t st = as_stream(stream);
  launch_attn(a, p, st);
  TB_LAUNCH_CHECK("paged_attn");
  if (!p.unit) {
    paged_join_kernel<<<dim3((unsigned)p.blocks, (unsigned)cdiv(p.R * D, 256)), kJoinWaves * 64, 0, st>>>(a);
    TB_LAUNCH_CHECK("paged_attn join");
  }
  return 0;
}
