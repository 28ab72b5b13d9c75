// A paged cache's bookkeeping on the device: sequences get longer and shorter, their pages come from
// a stack of free pages and go back to it, and every new token gets its slot and its position.
//
// With old lengths l, counts c, page the positions of a page, and e = max(0, l + min(c, 0)):
//   given back   table entries ceil(e / page) .. ceil(l / page), the last sequence's last entry first, so
//                that taking tokens back puts the stack as it was before they came (ids on it that are no page
//                aside, and table entries that were other than -1 past a sequence's pages); entries that name
//                no page are left out;
//   granted      sequence b with c > 0 where e + c fits its table row, the sum of c up to b is at most
//                `tokens`, and it needs no page or the sum of needs up to b is at most the free pages. Needs
//                of sequences that are not granted count as well, so the rule is two prefix sums.
// All granted sequences that need pages come before the first that lacks them, so the pages taken are a
// run of the stack from its top: the p-th new page of b is free[top - 1 - (needs before b) - p]. A
// token finds its page there by itself, and the page's first token writes the table entry.
//
// Nothing here is bound by memory or arithmetic: a chain of dependent steps (lengths, sums over the
// batch, search, page id) of about a microsecond each, 3.5 us in all for 64 sequences; 32 prompts of 65536 tokens
// together take 9.9.
#include <algorithm>
#include <type_traits>

#include "abi_util.h"
#include "common.h"

using namespace tbf16;

namespace {

struct AdvanceArgs {
  int32_t* table;
  int64_t t_sb;
  int B, n, cap;  // cap: positions the n entries of a table row cover
  int32_t* lengths;
  const int32_t* counts;
  int32_t* free;
  int P;
  int32_t* n_free;
  int page, tokens;
  const int32_t* prefix;
  int32_t *slots, *positions, *starts;
  // workspace: the free pages before any are taken; per sequence the length its new tokens begin at
  // (-1: none granted), the needs before it, the entries given back before it
  int32_t *top, *base, *first, *rel;
};

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Inclusive prefix sums over the wave, saturating (DPP row_shr 1, 2, 4, 8, row_bcast 15 and 31).
__device__ __forceinline__ uint32_t prefix_sat(uint32_t v) {
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return v;
}

// The last index i of the ascending v[0..n) with v[i] <= x (v[0] <= x).
__device__ __forceinline__ int last_upto(const int32_t* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// What a sequence wants: its old length, the length after giving back, new tokens and pages.
struct Want {
  int held, less;
  uint32_t more, need;
  bool fits;
};
__device__ __forceinline__ int pages_of(const AdvanceArgs& a, int len) { return (int)(((int64_t)len + a.page - 1) / a.page); }
__device__ __forceinline__ Want want(const AdvanceArgs& a, int b) {
  Want w;
  w.held = min(max(a.lengths[b], 0), a.cap);
  const int c = a.counts[b];
  w.less = c < 0 ? (int)max((int64_t)w.held + c, (int64_t)0) : w.held;
  w.more = (uint32_t)max(c, 0);
  w.fits = (int64_t)w.less + w.more <= a.cap;
  w.need = w.fits ? pages_of(a, w.less + (int)w.more) - pages_of(a, w.less) : 0;
  return w;
}

// Slot and position of token t, with starts, base and first wherever they are. (Several tokens a thread with
// their loads under way together were 0.7 us slower at 2000 and at 4000 tokens.)
__device__ __forceinline__ void token(const AdvanceArgs& a, int t, const int32_t* starts, const int32_t* base,
                                      const int32_t* first, int top, int prefix) {
  int slot = -1, pos = -1;
  if (a.B > 0 && t < starts[a.B]) {
    const int b = last_upto(starts, a.B, t), from = base[b];
    if (from >= 0) {
      // (unsigned, and with bounds that hold by themselves unless another stream writes lengths or counts meanwhile:
      // then from may be of one length and t - starts[b] of another's tokens, up to 2^32 together)
      const uint32_t j = (uint32_t)from + (uint32_t)(t - starts[b]), p = j / (uint32_t)a.page, r = j - p * (uint32_t)a.page;
      const uint32_t kept = (uint32_t)pages_of(a, from), at = (uint32_t)(top - 1 - first[b]) - (p - kept);
      int id = -1;
      if (p < min(kept, (uint32_t)a.n)) {
        id = a.table[b * a.t_sb + p];
      } else if (p < (uint32_t)a.n && at < (uint32_t)a.P) {
        id = a.free[at];
        if (r == 0) a.table[b * a.t_sb + p] = id;
      }
      if ((uint32_t)id < (uint32_t)a.P) slot = id * a.page + (int)r;
      pos = (int)min((int64_t)j + prefix, (int64_t)INT32_MAX);
    }
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

__device__ __forceinline__ int prefix_of(const AdvanceArgs& a) { return a.prefix ? max(*a.prefix, 0) : 0; }

// One block does everything but, with TOKENS false, the tokens: up to kInside of them cost it no more than a second
// launch does (device time of a call and of taking its tokens back, the mean: 2000 tokens 6.2 us, in a launch of
// their own 6.8; 4000: 7.4 and 6.8; 8000: 9.8 and 6.9). HERE: the batch's sums are kept in LDS (2000 sequences:
// 9.0 us, in memory 10.5), as far as it goes.
constexpr int kHere = 2048, kInside = 2048;
template <bool HERE, bool TOKENS>
__global__ __launch_bounds__(1024) void paged_advance_kernel(AdvanceArgs a) {
  __shared__ int32_t s_mem[HERE ? 4 * kHere + 4 : 1];
  __shared__ uint32_t s_wave[3][16];
  __shared__ uint32_t s_real[4][16];
  __shared__ uint32_t s_taken;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = nt >> 6;
  int32_t* const starts = HERE ? s_mem : a.starts;
  int32_t* const base = HERE ? s_mem + kHere + 1 : a.base;
  int32_t* const first = HERE ? base + kHere : a.first;
  int32_t* const rel = HERE ? first + kHere : a.rel;
  const int prefix = prefix_of(a);
  int top = min(max(*a.n_free, 0), a.P);
  if (tid == 0) s_taken = 0;

  // sums over the batch: tokens, needs, entries given back
  uint32_t sum_more = 0, sum_need = 0, sum_rel = 0;
  for (int b0 = 0; b0 < a.B; b0 += nt) {
    const int b = b0 + tid;
    Want w{0, 0, 0, 0, false};
    if (b < a.B) w = want(a, b);
    const uint32_t gone = pages_of(a, w.held) - pages_of(a, w.less);
    uint32_t up[3] = {prefix_sat(w.more), prefix_sat(w.need), prefix_sat(gone)};
    if (lane == 63)
#pragma unroll
      for (int i = 0; i < 3; ++i) s_wave[i][wave] = up[i];
    __syncthreads();
    uint32_t before[3] = {sum_more, sum_need, sum_rel};
    for (int v = 0; v < waves; ++v)
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const uint32_t s = s_wave[i][v];
        if (v < wave) before[i] = add_sat(before[i], s);
        if (i == 0) sum_more = add_sat(sum_more, s);
        if (i == 1) sum_need = add_sat(sum_need, s);
        if (i == 2) sum_rel = add_sat(sum_rel, s);
      }
    if (b < a.B) {
      const uint32_t ends = add_sat(before[0], up[0]);
      starts[b + 1] = (int)min(ends, (uint32_t)a.tokens);
      if (b == 0) starts[0] = 0;
      base[b] = w.less;
      // needs up to b and its own, for now; -1: not granted
      first[b] = ends > (uint32_t)a.tokens ? -1 : (int)min(add_sat(before[1], up[1]), (uint32_t)INT32_MAX);
      rel[b] = (int)(add_sat(before[2], up[2]) - gone);
    }
    __syncthreads();
  }
  if (a.B == 0 && tid == 0) starts[0] = 0;

  // entries given back, from the last one on
  if (sum_rel) {
    uint32_t pushed = 0;
    // (entries a thread has under way: one for few; four where ~4000 pages come and go, 10.4 -> 9.7 us as above)
    auto give_back = [&](auto under_way) {
      constexpr int U = decltype(under_way)::value;
      for (uint32_t i0 = 0; i0 < sum_rel; i0 += U * nt) {
        int id[U];
        int32_t* entry[U];
        uint64_t real[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t i = i0 + u * nt + tid;
          id[u] = -1;
          entry[u] = nullptr;
          if (i >= sum_rel) continue;
          const int at = (int)(sum_rel - 1 - i), b = last_upto(rel, a.B, at);
          entry[u] = a.table + b * a.t_sb + pages_of(a, base[b]) + (at - rel[b]);
          id[u] = *entry[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (entry[u]) *entry[u] = -1;
          real[u] = __ballot((uint32_t)id[u] < (uint32_t)a.P);
          if (lane == 0) s_real[u][wave] = __popcll(real[u]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
          uint32_t before = pushed;
          for (int v = 0; v < waves; ++v) {
            if (v < wave) before += s_real[u][v];
            pushed += s_real[u][v];
          }
          const uint32_t at = top + before + __popcll(real[u] & ((1ull << lane) - 1));
          if ((real[u] >> lane & 1) && at < (uint32_t)a.P) a.free[at] = id[u];
        }
        __syncthreads();
      }
    };
    if (sum_rel <= (uint32_t)nt) give_back(std::integral_constant<int, 1>());
    else give_back(std::integral_constant<int, 4>());
    top = (int)min((uint32_t)top + pushed, (uint32_t)a.P);
  }

  // who gets tokens
  for (int b = tid; b < a.B; b += nt) {
    const Want w = want(a, b);
    const int upto = first[b];
    const bool ok = w.more > 0 && w.fits && upto >= 0 && (w.need == 0 || upto <= top);
    a.lengths[b] = ok ? w.less + (int)w.more : w.less;
    base[b] = ok ? w.less : -1;
    first[b] = upto - (int)w.need;
    if (ok && w.need) atomicMax(&s_taken, (uint32_t)upto);
  }
  __syncthreads();
  if (tid == 0) *a.n_free = top - (int)s_taken;
  if constexpr (HERE)
    for (int b = tid; b <= a.B; b += nt) a.starts[b] = starts[b];
  if constexpr (TOKENS) {
    for (int t = tid; t < a.tokens; t += nt) token(a, t, starts, base, first, top, prefix);
  } else {
    if (tid == 0) *a.top = top;
    if constexpr (HERE)
      for (int b = tid; b < a.B; b += nt) {
        a.base[b] = base[b];
        a.first[b] = first[b];
      }
  }
}

__global__ __launch_bounds__(256) void paged_tokens_kernel(AdvanceArgs a) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < a.tokens) token(a, t, a.starts, a.base, a.first, *a.top, prefix_of(a));
}

}  // namespace

extern "C" size_t tbf16_paged_advance_ws_bytes(int64_t B, int64_t tokens) {
  return B < 0 ? 0 : B <= kHere && tokens <= kInside ? 0 : (size_t)(3 * B + 4) * 4;
}

extern "C" int tbf16_paged_advance(int32_t* table, int64_t table_stride, int64_t B, int64_t max_pages, int32_t* lengths,
                                   const int32_t* counts, int32_t* free_pages, int64_t pages, int32_t* n_free, int64_t page,
                                   int64_t tokens, const int32_t* prefix, int32_t* slots, int32_t* positions,
                                   int32_t* starts, void* ws, int64_t ws_bytes, void* stream) {
  const int64_t top31 = (int64_t)1 << 31;
  TB_CHECK(B >= 0 && B < top31 / 2 && max_pages >= 0 && max_pages < top31 && (double)B * (double)max_pages < 2147483648.0,
           "paged_advance: bad table shape");
  TB_CHECK(B <= 1 || table_stride >= max_pages, "paged_advance: table rows overlap");
  TB_CHECK(page > 0 && page < top31 && pages >= 0 && (double)pages * (double)page < 2147483647.0,
           "paged_advance: more slots than int32 counts");
  TB_CHECK(tokens >= 0 && tokens < top31 - 1024, "paged_advance: bad number of tokens");
  for (const void* p : {(const void*)table, (const void*)lengths, (const void*)counts, (const void*)free_pages,
                        (const void*)n_free, (const void*)prefix, (const void*)slots, (const void*)positions,
                        (const void*)starts, (const void*)ws})
    TB_CHECK(aligned4(p), "paged_advance: misaligned pointer");
  TB_CHECK(n_free != nullptr && starts != nullptr, "paged_advance: missing pointer");
  const size_t need = tbf16_paged_advance_ws_bytes(B, tokens);
  if (ws_bytes < (int64_t)need || (need && ws == nullptr)) {
    set_error("paged_advance: workspace too small (%lld bytes, needs %zu)", (long long)ws_bytes, need);
    return TBF16_EWS;
  }
  AdvanceArgs a = {};
  a.table = table;
  a.t_sb = table_stride;
  a.B = (int)B;
  a.n = (int)max_pages;
  a.cap = (int)std::min<int64_t>(max_pages * page, INT32_MAX);
  a.lengths = lengths;
  a.counts = counts;
  a.free = free_pages;
  a.P = (int)pages;
  a.n_free = n_free;
  a.page = (int)page;
  a.tokens = (int)tokens;
  a.prefix = prefix;
  a.slots = slots;
  a.positions = positions;
  a.starts = starts;
  if (need) {
    a.top = (int32_t*)ws;
    a.base = a.top + 4;
    a.first = a.base + B;
    a.rel = a.first + B;
  }
  const hipStream_t st = as_stream(stream);
  const bool here = B <= kHere, inside = tokens <= kInside;
  // Few waves meet sooner at barriers (as above; 64 sequences, 6 tokens: 512 threads 3.5 us, 1024 4.2; 512 sequences,
  // a token each: 4.9 and 5.7; 2000: 10.9 and 9.0).
  const int nt = std::max(B, inside ? tokens : 0) <= 1024 ? 512 : 1024;
  if (here && inside) paged_advance_kernel<true, true><<<1, nt, 0, st>>>(a);
  else if (here) paged_advance_kernel<true, false><<<1, nt, 0, st>>>(a);
  else if (inside) paged_advance_kernel<false, true><<<1, nt, 0, st>>>(a);
  else paged_advance_kernel<false, false><<<1, nt, 0, st>>>(a);
  TB_LAUNCH_CHECK("paged_advance");
  if (!inside) {
    paged_tokens_kernel<<<(unsigned)cdiv(tokens, 256), 256, 0, st>>>(a);
    TB_LAUNCH_CHECK("paged_advance tokens");
  }
  return 0;
}
