// A paged key/value cache: writing new tokens into it, and attention of one new token per
// sequence over it.
//
// The cache is two bf16 tensors (pages, Hkv, page, D): position j of sequence b lives in
// page table[b][j / page], row j % page. The entry points take element strides, so other
// orders of the same axes work as views.
#include <float.h>

#include <algorithm>

#include "abi_util.h"
#include "common.h"

using namespace tbf16;

namespace {

struct CacheGeom {
  int64_t sp, sh, ss;  // element strides of page, head and row
};

// ---- write ------------------------------------------------------------------------

// One wave per token: its 16-byte chunks of all heads, keys then values. A slot that a
// later token names too is left to that token, so a repeated slot holds the last one's
// whole row whatever the order of the waves.
__global__ __launch_bounds__(256) void paged_write_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                          int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                                                          const int32_t* __restrict__ slots, int T, int Hkv, int D8,
                                                          uint16_t* __restrict__ kc, uint16_t* __restrict__ vc,
                                                          CacheGeom kg, CacheGeom vg, int64_t n_slots, int page) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= T) return;
  const int slot = slots[t];
  if (slot < 0 || slot >= n_slots) return;
  for (int u = t + 1 + lane; __any(u < T); u += 64)
    if (__any(u < T && slots[u] == slot)) return;
  const int64_t p = slot / page, r = slot % page;
  for (int i = lane; i < Hkv * D8; i += 64) {
    const int h = i / D8, c = i % D8 * 8;
    stg16(kc + p * kg.sp + h * kg.sh + r * kg.ss + c, ldg16(k + t * k_st + h * k_sh + c));
    stg16(vc + p * vg.sp + h * vg.sh + r * vg.ss + c, ldg16(v + t * v_st + h * v_sh + c));
  }
}

// ---- attention ----------------------------------------------------------------------

// One block per (sequence, query head): 256 keys at a time, a thread per key for the
// logits, a thread per output element for the weighted sum. Running maximum and sum in
// fp32 (log2 domain).
__global__ __launch_bounds__(256) void paged_attn_kernel(const uint16_t* __restrict__ q, int64_t q_sb, int64_t q_sh,
                                                         const uint16_t* __restrict__ kc, const uint16_t* __restrict__ vc,
                                                         CacheGeom kg, CacheGeom vg, int64_t pages, int page,
                                                         const int32_t* __restrict__ table, int64_t t_sb, int max_pages,
                                                         const int32_t* __restrict__ lengths, float scale_log2, int H,
                                                         int G, int D, uint16_t* __restrict__ o) {
  __shared__ float qs[256], w[256], red[4];
  __shared__ int64_t row[256];
  const int b = blockIdx.x / H, h = blockIdx.x % H, tid = threadIdx.x;
  const int64_t cap = (int64_t)max_pages * page;
  const int len = (int)min<int64_t>(max(lengths[b], 0), cap);
  if (tid < D) qs[tid] = bf16_lo(q[b * q_sb + h * q_sh + tid]);
  __syncthreads();
  // the lowest finite value: infinite logits below it weigh nothing, and nothing is inf - inf
  float m = -FLT_MAX, l = 0.f, acc = 0.f;
  bool some = false;
  for (int j0 = 0; j0 < len; j0 += 256) {
    const int j = j0 + tid;
    float s = -INFINITY;
    int64_t at = -1;
    if (j < len) {
      const int p = table[b * t_sb + j / page];
      if (p >= 0 && p < pages) {
        at = p;
        const uint16_t* kr = kc + p * kg.sp + (h / G) * kg.sh + (j % page) * kg.ss;
        s = 0.f;
        for (int d = 0; d < D; ++d) s = fmaf(qs[d], bf16_lo(kr[d]), s);
        s *= scale_log2;
      }
    }
    row[tid] = at;
    float mt = wave_max(s);
    if ((tid & 63) == 0) red[tid >> 6] = mt;
    const bool here = __syncthreads_or(at >= 0);
    if (here) {
      some = true;
      // a NaN logit has to reach the output: the maximum may leave it out, its weight is NaN
      const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
      const float f = exp2f(m - mn);
      w[tid] = at >= 0 ? exp2f(s - mn) : 0.f;
      __syncthreads();
      acc *= f;
      l *= f;
      for (int i = 0; i < 256; ++i)
        if (row[i] >= 0) {
          l += w[i];
          if (tid < D)
            acc = fmaf(w[i], bf16_lo(vc[row[i] * vg.sp + (h / G) * vg.sh + ((j0 + i) % page) * vg.ss + tid]), acc);
        }
      m = mn;
    }
    __syncthreads();
  }
  if (tid < D) {
    const float y = some ? acc / l : 0.f;
    o[((int64_t)b * H + h) * D + tid] = (uint16_t)pack_bf16(y, 0.f);
  }
}

int check_cache(const char* fn, const void* kc, const void* vc, int64_t pages, int64_t Hkv, int64_t page, int64_t D,
                const int64_t* ks, const int64_t* vs) {
  TB_CHECK(pages >= 0 && Hkv > 0 && page > 0 && D > 0, "%s: bad cache shape", fn);
  TB_CHECK(pages < (int64_t)1 << 31 && page < (int64_t)1 << 31 && Hkv < (int64_t)1 << 20, "%s: cache too large", fn);
  TB_CHECK(D % 8 == 0, "%s: head dim must be a multiple of 8", fn);
  TB_CHECK(aligned16(kc) && aligned16(vc), "%s: cache must be 16-byte aligned", fn);
  for (int i = 0; i < 3; ++i)
    TB_CHECK(ks[i] % 8 == 0 && vs[i] % 8 == 0 && ks[i] >= 0 && vs[i] >= 0 && ks[i] < (int64_t)1 << 31 && vs[i] < (int64_t)1 << 31,
             "%s: cache strides must be multiples of 8 below 2^31", fn);
  return 0;
}

}  // namespace

extern "C" int tbf16_paged_write(const void* k, const void* v, int64_t T, int64_t Hkv, int64_t D, const int64_t* k_strides,
                                 const int64_t* v_strides, const int32_t* slots, void* k_cache, void* v_cache,
                                 int64_t pages, int64_t page, const int64_t* kc_strides, const int64_t* vc_strides,
                                 void* stream) {
  if (int rc = check_cache("paged_write", k_cache, v_cache, pages, Hkv, page, D, kc_strides, vc_strides)) return rc;
  TB_CHECK(T >= 0 && T < (int64_t)1 << 31, "paged_write: bad number of tokens");
  TB_CHECK(aligned16(k) && aligned16(v) && aligned4(slots), "paged_write: k and v must be 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    TB_CHECK(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, "paged_write: strides must be multiples of 8");
  if (T == 0 || pages == 0) return 0;
  paged_write_kernel<<<(unsigned)cdiv(T, 4), 256, 0, as_stream(stream)>>>(
      (const uint16_t*)k, (const uint16_t*)v, k_strides[0], k_strides[1], v_strides[0], v_strides[1], slots, (int)T,
      (int)Hkv, (int)(D / 8), (uint16_t*)k_cache, (uint16_t*)v_cache, CacheGeom{kc_strides[0], kc_strides[1], kc_strides[2]},
      CacheGeom{vc_strides[0], vc_strides[1], vc_strides[2]}, pages * page, (int)page);
  TB_LAUNCH_CHECK("paged_write");
  return 0;
}

extern "C" size_t tbf16_paged_attn_ws_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D) {
  return B > 0 && H > 0 && Hkv > 0 && D > 0 ? 16 : 0;
}

extern "C" int tbf16_paged_attn(const void* q, int64_t B, int64_t H, int64_t Hkv, int64_t D, const int64_t* q_strides,
                                const void* k_cache, const void* v_cache, int64_t pages, int64_t page,
                                const int64_t* kc_strides, const int64_t* vc_strides, const int32_t* table,
                                int64_t table_stride, int64_t max_pages, const int32_t* lengths, float scale, void* o,
                                void* ws, int64_t ws_bytes, void* stream) {
  TB_CHECK(B >= 0 && H > 0, "paged_attn: bad shape");
  if (int rc = check_cache("paged_attn", k_cache, v_cache, pages, Hkv, page, D, kc_strides, vc_strides)) return rc;
  TB_CHECK(H % Hkv == 0, "paged_attn: query heads must be a multiple of key/value heads");
  TB_CHECK(D <= 256, "paged_attn: head dim must be at most 256");
  TB_CHECK(B * H < (int64_t)1 << 31 && max_pages >= 0 && max_pages < (int64_t)1 << 31, "paged_attn: shape too large");
  TB_CHECK(aligned16(q) && aligned16(o) && q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0,
           "paged_attn: q must have 16-byte aligned rows");
  TB_CHECK(aligned4(table) && aligned4(lengths), "paged_attn: table and lengths must be 4-byte aligned");
  if (B == 0) return 0;
  TB_CHECK(aligned16(ws) && ws != nullptr, "paged_attn: workspace missing or misaligned");
  if (ws_bytes < (int64_t)tbf16_paged_attn_ws_bytes(B, H, Hkv, D)) {
    set_error("paged_attn: workspace too small");
    return TBF16_EWS;
  }
  paged_attn_kernel<<<(unsigned)(B * H), 256, 0, as_stream(stream)>>>(
      (const uint16_t*)q, q_strides[0], q_strides[1], (const uint16_t*)k_cache, (const uint16_t*)v_cache,
      CacheGeom{kc_strides[0], kc_strides[1], kc_strides[2]}, CacheGeom{vc_strides[0], vc_strides[1], vc_strides[2]}, pages,
      (int)page, table, table_stride, (int)max_pages, lengths, scale * 1.4426950408889634f, (int)H, (int)(H / Hkv), (int)D,
      (uint16_t*)o);
  TB_LAUNCH_CHECK("paged_attn");
  return 0;
}
