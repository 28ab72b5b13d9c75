// Attention of one new token per sequence over a paged cache where all sequences begin with the same
// tokens: the prefix's keys and values are read once for the whole batch.
//
// o = softmax of the logits of prefix keys and own keys together, times their values. Any split of the keys into
// parts gives (m, l, o) with o = sum_j 2^(x_j - m) v_j and l = sum_j 2^(x_j - m), and parts join as
//   m = max m_i,   l = sum l_i 2^(m_i - m),   o = sum o_i 2^(m_i - m).
// Three launches: the prefix (prefix_kernel), the sequences' own keys (paged_attn_kernel of paged_attn.h, which
// leaves sums instead of outputs), the join of all parts of a row (prefix_join_kernel).
#include "paged_attn.h"

using namespace tbf16;

namespace {

struct PrefixArgs {
  const uint16_t *q, *kc, *vc;
  int64_t q_sb, q_sh;
  CacheGeom kg, vg;
  const int32_t *table, *length;
  int cap, S;  // positions the table covers; splits of the keys
  uint32_t pages, page;
  Div by_page, by_group;
  float scale_log2;
  int B, H, Hkv, G, D;
  float *part, *stat;  // [split][b H + h][D], [split][b H + h][2]
};

__device__ const uint4 kZeros = {0, 0, 0, 0};

// Which tiles a split takes, of `keys` positions each: equal runs, the last ones may have none.
struct Splits {
  int tiles, each;
};
__device__ __forceinline__ Splits splits_of(int length, int keys, int S) {
  const int tiles = (int)(((int64_t)length + keys - 1) / keys);
  return {tiles, max(1, (tiles + S - 1) / S)};
}
__device__ __forceinline__ int prefix_len(const int32_t* length, int cap) { return min(max(uniform(*length), 0), cap); }

// ---- the prefix -------------------------------------------------------------------------
//
// A product of many rows with the prefix's keys: rows r = 0 .. B G - 1 of a key/value head are query
// head head G + r % G of sequence r / G. NW = WR WK waves a block; a wave has RB blocks of 16
// rows, WR of them side by side; WK groups of waves take different keys of a stage and are joined at the
// end. A stage is KS = 32 KB WK keys of K and V, row-major in LDS, filled by direct loads from wherever the
// page table says (each lane its own address), ST stages in a ring.
//
// S^T = K Q^T on v_mfma_f32_16x16x32_bf16: lane l gets keys 4 (l / 16) .. + 3 of each 16-key block for row l % 16,
// which are its k slots of O^T = V^T P^T; V^T comes from the row-major tile by ds_read_b64_tr_b16. The maximum a
// row's weights refer to follows its largest logit only in steps of 2^8 (weights then reach 2^8 of the last
// step's; they carry 2^-16, so that sums have the room that paged_attn.h's have). Weights go into the second product as
// the sum of two bf16: 8 bits, and the next 9 rounded to nearest.
//
// LDS: chunk c of 16 bytes of row r lies at chunk c ^ f(r) of its row, so that the 16 rows that a read of
// K takes at one chunk lie in all 64 banks, and so do the two chunks of 8 rows that a transposed read takes.
template <int DP>
__device__ __forceinline__ int swz(int row) {
  if constexpr (DP >= 128) return ((row & 7) << 1) | ((row >> 3) & 1);
  else return (((row >> 1) & 3) << 1) | ((row >> 3) & 1);
}

constexpr int kIds = 4096;  // page ids a block holds at a time
constexpr float kLag = 8.f;

typedef __attribute__((address_space(1))) void global_void;
__device__ __forceinline__ void load16_lds(const void* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((global_void*)from, (lds_void*)to, 16, 0, 0);
}

template <int DP, int RB, int WR, int WK, int KB, int ST, bool PAD>
__global__ __launch_bounds__(WR * WK * 64, 1) void prefix_kernel(PrefixArgs a) {
  constexpr int NW = WR * WK, KS = 32 * KB * WK, CPR = DP / 8, RPI = 64 / CPR;  // chunks of a row, rows of a load
  constexpr int KPW = KS / RPI / NW;                                             // loads of K a wave does for a stage
  constexpr int KBYTES = KS * DP * 2, STAGE = 2 * KBYTES, KI = DP / 32, DB = DP / 16;
  static_assert(KS % (RPI * NW) == 0 && ST >= 2 && ST <= 4 && (ST - 2) * 2 * KPW < 63, "stage shape");
  __shared__ __align__(1024) uint8_t st0[STAGE], st1[STAGE], st2[ST > 2 ? STAGE : 16], st3[ST > 3 ? STAGE : 16];
  __shared__ int s_ids[kIds];
  __shared__ float2 s_stat[NW][16 * RB];
  uint8_t* const stages[4] = {st0, st1, st2, st3};
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r16 = lane & 15;
  const int wr = wave % WR, kg = wave / WR;
  const int head = blockIdx.x % a.Hkv, split = blockIdx.x / a.Hkv % a.S, rt = blockIdx.x / a.Hkv / a.S;
  const int length = prefix_len(a.length, a.cap);
  const Splits sp = splits_of(length, KS, a.S);
  const int t0 = split * sp.each, tn = min(sp.each, sp.tiles - t0);
  if (tn <= 0) return;

  // the wave's rows
  const int rows = a.B * a.G, row0 = (rt * WR + wr) * 16 * RB;
  const float c = fabsf(a.scale_log2);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  bf16x8 qf[RB][KI];
  int64_t out[RB];  // the lane's rows' place in the parts, -1: none
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = row0 + 16 * r + r16, b = min(row, rows - 1) / a.by_group, h = head * a.G + min(row, rows - 1) - b * a.G;
    out[r] = row < rows ? ((int64_t)split * a.B + b) * a.H + h : -1;
    const uint16_t* src = a.q + b * a.q_sb + h * a.q_sh;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int e = 8 * (g + 4 * i);
      uint4 v = ldg16(src + (!PAD || e < a.D ? e : 0));
      if (PAD && e >= a.D) v = make_uint4(0, 0, 0, 0);
      qf[r][i] = __builtin_bit_cast(bf16x8, make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip));
    }
  }

  floatx4 o[RB][DB];
  float m[RB], l[RB];  // m: what the weights refer to
  bool fresh = true;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m[r] = kNone;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[r][d] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  const uint16_t *kc = a.kc + head * a.kg.sh, *vc = a.vc + head * a.vg.sh;
  int id0 = 0;  // the first page whose id s_ids holds
  // id of the page of position pos, -1 past the prefix's end
  auto page_of = [&](int pos, int& row) {
    const uint32_t at = min(pos, length - 1), idx = at / a.by_page;
    row = (int)(at - idx * a.page);
    const int id = s_ids[(int)idx - id0];
    return pos < length && (uint32_t)id < a.pages ? id : -1;
  };
  const int lrow = lane / CPR, lchunk = lane % CPR;
  auto issue = [&](uint8_t* stage, int tile) {
#pragma unroll
    for (int j = 0; j < KPW; ++j) {
      const int n = wave * KPW + j, krow = n * RPI + lrow, chunk = lchunk ^ swz<DP>(krow);
      int row;
      const int id = page_of(tile * KS + krow, row);
      const bool there = id >= 0 && (!PAD || chunk * 8 < a.D);
      const uint16_t* k = kc + (int64_t)id * a.kg.sp + (int64_t)row * a.kg.ss + chunk * 8;
      const uint16_t* v = vc + (int64_t)id * a.vg.sp + (int64_t)row * a.vg.ss + chunk * 8;
      load16_lds(there ? (const void*)k : &kZeros, stage + n * 1024);
      load16_lds(there ? (const void*)v : &kZeros, stage + KBYTES + n * 1024);
    }
  };

  // the lane's place in fragments: K row r16, chunk g (+ 4 t); V^T keys 4 g + r16 / 4, columns 4 (r16 % 4)
  const int klane = (kg * 32 * KB + r16) * DP * 2 + ((g ^ swz<DP>(r16)) << 4);
  const int vrow = 4 * g + (r16 >> 2);
  const int vlane = KBYTES + (kg * 32 * KB + vrow) * DP * 2 + (((r16 & 3) >> 1 ^ swz<DP>(vrow)) << 4) + 8 * (r16 & 1);
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lds_v4s;

  auto compute = [&](const uint8_t* stage, int tile) {
    int unused;
    const int key = lane & (32 * KB - 1);
    uint64_t live = __ballot(page_of(tile * KS + kg * 32 * KB + key, unused) >= 0);
    if constexpr (KB == 1) live &= 0xffffffffu;
    if (live == 0) return;
    const bool whole = live == (KB == 1 ? 0xffffffffull : ~0ull);
    floatx4 s[2 * KB][RB];
#pragma unroll
    for (int k = 0; k < 2 * KB; ++k)
#pragma unroll
      for (int r = 0; r < RB; ++r) s[k][r] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KI; ++t)
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k) {
        const bf16x8 kf = *reinterpret_cast<const bf16x8*>(stage + (klane ^ (t << 6)) + k * 16 * DP * 2);
#pragma unroll
        for (int r = 0; r < RB; ++r) s[k][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[r][t], s[k][r], 0, 0, 0);
      }
    float cc = c;
    if (!whole) {
      cc = 1.f;
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[k][r][i] = live >> (16 * k + 4 * g + i) & 1 ? s[k][r][i] * c : -INFINITY;
    }
    float mx[RB];
    bool grown = fresh;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      mx[r] = -INFINITY;
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[r] = fmaxf(mx[r], s[k][r][i]);
      mx[r] *= cc;
      grown |= mx[r] > m[r] + kLag;
    }
    if (__any(grown)) {
      fresh = false;
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float mn = fmaxf(mx[r], kFew);
        mn = fmaxf(mn, __shfl_xor(mn, 16, kWave));
        mn = fmaxf(mn, __shfl_xor(mn, 32, kWave));
        mn = fmaxf(mn, m[r]);
        const float f = ex2(m[r] - mn);
        m[r] = mn;
        l[r] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[r][d] *= f;
      }
    }
#pragma unroll
    for (int h = 0; h < KB; ++h) {  // 32 keys
      bf16x8 pf[RB][2];
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float mo = m[r] + 2 * kLag;
        uint32_t f[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const floatx4& sv = s[2 * h + (j >> 1)][r];
          const float p0 = ex2(fmaf(sv[2 * (j & 1)], cc, -mo)), p1 = ex2(fmaf(sv[2 * (j & 1) + 1], cc, -mo));
          l[r] += p0 + p1;
          f[0][j] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302u);
          f[1][j] = pack_bf16(p0 - bf16_hi(__float_as_uint(p0)), p1 - bf16_hi(__float_as_uint(p1)));
          // 2^-28 of p in place of a part that is zero: an infinite value times it stays infinite
          const ushort2v least = __builtin_elementwise_sub_sat(__builtin_bit_cast(ushort2v, f[0][j]), ushort2v{28 << 7, 28 << 7});
          f[1][j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, f[1][j]), least));
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) pf[r][t] = __builtin_bit_cast(bf16x8, make_uint4(f[t][0], f[t][1], f[t][2], f[t][3]));
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const uint8_t* at = stage + (vlane ^ (d << 5)) + h * 32 * DP * 2;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 16 * DP * 2));
        const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t) o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[r][t], o[r][d], 0, 0, 0);
      }
    }
  };

  // as many tiles at a time as s_ids covers
  const int most = (int)min((int64_t)tn, max((int64_t)1, (int64_t)(kIds - 2) * a.page / KS));
  for (int done = 0; done < tn; done += most) {
    const int first = t0 + done, n = min(most, tn - done);
    const int from = first * KS, last = min(from + n * KS, length) - 1;
    __syncthreads();  // nobody reads the ids or stages of the tiles before
    id0 = (int)((uint32_t)from / a.by_page);
    const int ids = (int)((uint32_t)last / a.by_page) - id0 + 1;
    for (int i = threadIdx.x; i < ids; i += NW * 64) s_ids[i] = a.table[id0 + i];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ST - 1; ++u)
      if (u < n) issue(stages[u], first + u);
    for (int i0 = 0; i0 < n; i0 += ST) {
#pragma unroll
      for (int u = 0; u < ST; ++u) {
        const int i = i0 + u;
        if (i >= n) break;
        // stage u is there once only the later stages' loads are on their way
        if (i + ST - 2 < n) wait_vmem_n<(ST - 2) * 2 * KPW>();
        else wait_vmem_n<0>();
        wait_lds();
        barrier_no_fence();
        if (i + ST - 1 < n) issue(stages[(u + ST - 1) % ST], first + i + ST - 1);
        compute(stages[u], first + i);
      }
    }
  }

#pragma unroll
  for (int r = 0; r < RB; ++r) l[r] = sum_xor32(sum_xor16(l[r]));
  if constexpr (WK > 1) {  // the groups' parts meet in the first one, through the stages' memory
    constexpr int PART = 16 * RB * DP * 4, PER = STAGE / PART;
    static_assert((WK - 1) * WR <= PER * ST, "parts fit the stages");
    __syncthreads();
    auto place = [&](int of) {  // of wave `of` of the later groups
      const int at = of / PER;
      return reinterpret_cast<floatx4*>((at == 0 ? st0 : at == 1 ? st1 : at == 2 ? st2 : st3) + of % PER * PART) + lane;
    };
    if (kg > 0) {
      floatx4* to = place((kg - 1) * WR + wr);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
#pragma unroll
        for (int d = 0; d < DB; ++d) to[(r * DB + d) * 64] = o[r][d];
        if (g == 0) s_stat[wave][16 * r + r16] = make_float2(m[r], l[r]);
      }
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float2 st[WK];
      float mn = m[r];
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        st[k] = s_stat[k * WR + wr][16 * r + r16];
        mn = fmaxf(mn, st[k].x);
      }
      const float f = ex2(m[r] - mn);
      m[r] = mn;
      l[r] *= f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[r][d] *= f;
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        const float h = ex2(st[k].x - mn);
        l[r] = fmaf(h, st[k].y, l[r]);
        const floatx4* from = place((k - 1) * WR + wr);
#pragma unroll
        for (int d = 0; d < DB; ++d) o[r][d] += h * from[(r * DB + d) * 64];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (out[r] < 0) continue;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const int at = 16 * d + 4 * g;
      if (!PAD || at < a.D) *reinterpret_cast<floatx4*>(a.part + out[r] * a.D + at) = o[r][d];
    }
    // (in the terms of paged_attn.h, whose weights are 2^(x - m - 8))
    if (g == 0) *reinterpret_cast<float2*>(a.stat + out[r] * 2) = make_float2(m[r] == kNone ? kNone : m[r] + kLag, l[r]);
  }
}

// ---- the join -----------------------------------------------------------------------------

struct JoinArgs {
  AttnArgs own;
  PrefixArgs pre;
  int keys;   // of a tile of the prefix
  bool unit;  // the own keys' sums are all in own.own
  int blocks;  // of the own keys' list
  uint16_t* o;
};

// 64 groups of 4 outputs a block; its waves take a row's parts in turns and meet in LDS.
constexpr int kMeet = 8;
__global__ __launch_bounds__(kMeet * 64) void prefix_join_kernel(JoinArgs j) {
  __shared__ float4 so[kMeet][64];
  __shared__ float2 ss[kMeet][64];
  const AttnArgs& a = j.own;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), dg = a.D / 4;
  const int64_t all = (int64_t)a.B * a.H, e = (int64_t)blockIdx.x * 64 + lane;
  const int64_t row = min(e / dg, all - 1);
  const int d = (int)(e % dg) * 4;
  float m = kNone, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 s, float4 v) {
    if (s.x == kNone) return;  // no key: nothing was put there
    const float mn = fmaxf(m, s.x), f = ex2(m - mn), h = ex2(s.x - mn);
    m = mn;
    l = fmaf(l, f, s.y * h);
    o.x = fmaf(o.x, f, v.x * h);
    o.y = fmaf(o.y, f, v.y * h);
    o.z = fmaf(o.z, f, v.z * h);
    o.w = fmaf(o.w, f, v.w * h);
  };
  constexpr int U = 4;  // parts in flight
  if (j.pre.S > 0) {
    const Splits sp = splits_of(prefix_len(j.pre.length, j.pre.cap), j.keys, j.pre.S);
    const int used = (sp.tiles + sp.each - 1) / sp.each;
    for (int i0 = wave; i0 < used; i0 += U * kMeet) {
      float2 s[U];
      float4 v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t at = min(i0 + k * kMeet, used - 1) * all + row;
        s[k] = *reinterpret_cast<const float2*>(j.pre.stat + at * 2);
        v[k] = *reinterpret_cast<const float4*>(j.pre.part + at * a.D + d);
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i0 + k * kMeet < used) add(s[k], v[k]);
    }
  }
  // own keys
  int2 at = make_int2(kHere, kHere);
  int r = 0;
  if (!j.unit) {
    const int b = (int)(row / a.H), h = (int)(row - (int64_t)b * a.H), head = h / a.G, in = h - head * a.G, grp = in / a.R;
    r = in - grp * a.R;
    at = a.where[((int64_t)b * a.Hkv + head) * a.RG + grp];
  }
  if (at.x == kHere) {
    if (wave == kMeet - 1)
      add(*reinterpret_cast<const float2*>(a.own_stat + row * 2), *reinterpret_cast<const float4*>(a.own + row * a.D + d));
  } else if (at.x >= 0 && at.x < j.blocks) {  // (elsewhere, if the lengths changed since)
    for (int i = at.x + wave; i <= min(at.y, j.blocks - 1); i += kMeet) {
      const int64_t slot = (int64_t)i * 2 + (i == at.x ? 1 : 0);
      add(*reinterpret_cast<const float2*>(a.stat + (slot * a.R + r) * 2),
          *reinterpret_cast<const float4*>(a.part + (slot * a.R + r) * a.D + d));
    }
  }
  so[wave][lane] = o;
  ss[wave][lane] = make_float2(m, l);
  __syncthreads();
  if (wave != 0 || e >= all * dg) return;
#pragma unroll
  for (int w = 1; w < kMeet; ++w) add(ss[w][lane], so[w][lane]);
  const float f = m == kNone ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(j.o + row * a.D + d) = make_uint2(pack_bf16(o.x * f, o.y * f), pack_bf16(o.z * f, o.w * f));
}

// ---- host -------------------------------------------------------------------------------

// How a call is split: rows of a block and keys of a tile by the form, splits of the prefix.
struct PrefixPlan {
  int DP, form, rows, keys;
  int64_t tiles, S;  // row tiles of a key/value head, splits
  AttnPlan own;
  size_t part, stat, own_part, own_stat, where, bytes;
};
PrefixPlan prefix_plan(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t prefix_cap, int64_t cap) {
  PrefixPlan p;
  const int64_t n = B * (H / Hkv);
  p.DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  if (p.DP == 256) {
    p.form = n <= 32 ? 2 : n <= 64 ? 1 : 0;
    p.rows = p.form == 2 ? 32 : p.form == 1 ? 64 : 128;
    p.keys = 64;
  } else {
    p.form = n <= 32 ? 3 : n <= 64 ? 2 : n <= 128 ? 1 : 0;
    p.rows = 256 >> p.form;
    p.keys = p.form >= 2 ? 128 : 64;
  }
  p.tiles = cdiv(n, p.rows);
  p.S = std::min(cdiv(prefix_cap, p.keys), std::max<int64_t>(1, num_cus() / (Hkv * p.tiles)));
  p.own = attn_plan(B, H, Hkv, D, cap);
  p.part = align_up(p.own.bytes, 256);
  p.stat = p.part + align_up((size_t)(p.S * B * H * D) * 4, 256);
  p.own_part = p.stat + align_up((size_t)(p.S * B * H) * 8, 256);
  p.own_stat = p.own_part + align_up((size_t)(B * H * D) * 4, 256);
  p.where = p.own_stat + align_up((size_t)(B * H) * 8, 256);
  p.bytes = p.where + align_up((size_t)(B * Hkv * p.own.RG) * 8, 256);
  return p;
}

template <int DP, int RB, int WR, int WK, int KB, int ST>
void launch_form(const PrefixArgs& a, const PrefixPlan& p, hipStream_t st) {
  const unsigned grid = (unsigned)(a.Hkv * p.S * p.tiles);
  if (a.D == DP) prefix_kernel<DP, RB, WR, WK, KB, ST, false><<<grid, WR * WK * 64, 0, st>>>(a);
  else prefix_kernel<DP, RB, WR, WK, KB, ST, true><<<grid, WR * WK * 64, 0, st>>>(a);
}
void launch_prefix(const PrefixArgs& a, const PrefixPlan& p, hipStream_t st) {
  if (p.DP == 64) {
    if (p.form == 0) launch_form<64, 2, 8, 1, 2, 4>(a, p, st);
    else if (p.form == 1) launch_form<64, 2, 4, 2, 1, 4>(a, p, st);
    else if (p.form == 2) launch_form<64, 2, 2, 4, 1, 4>(a, p, st);
    else launch_form<64, 2, 1, 4, 1, 4>(a, p, st);
  } else if (p.DP == 128) {
    if (p.form == 0) launch_form<128, 2, 8, 1, 2, 4>(a, p, st);
    else if (p.form == 1) launch_form<128, 2, 4, 2, 1, 4>(a, p, st);
    else if (p.form == 2) launch_form<128, 2, 2, 4, 1, 2>(a, p, st);
    else launch_form<128, 2, 1, 4, 1, 2>(a, p, st);
  } else {
    if (p.form == 0) launch_form<256, 1, 8, 1, 2, 2>(a, p, st);
    else if (p.form == 1) launch_form<256, 1, 4, 2, 1, 2>(a, p, st);
    else launch_form<256, 1, 2, 2, 1, 2>(a, p, st);
  }
}

bool sizes_ok(int64_t B, int64_t H, int64_t Hkv, int64_t D) {
  return B > 0 && H > 0 && Hkv > 0 && D > 0 && D <= 256 && H % Hkv == 0 && H < (int64_t)1 << 24 &&
         (double)B * (double)H < 1e9;
}

}  // namespace

extern "C" size_t tbf16_paged_attn_prefix_ws_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t prefix_positions,
                                                   int64_t positions) {
  return sizes_ok(B, H, Hkv, D) && prefix_positions >= 0 && positions >= 0
             ? prefix_plan(B, H, Hkv, D, prefix_positions, positions).bytes
             : 0;
}

extern "C" int tbf16_paged_attn_prefix(const void* q, int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t q_sb, int64_t q_sh,
                                       const void* k_cache, const void* v_cache, int64_t pages, int64_t page, int64_t kc_sp,
                                       int64_t kc_sh, int64_t kc_ss, int64_t vc_sp, int64_t vc_sh, int64_t vc_ss,
                                       const int32_t* prefix_table, int64_t prefix_pages, const int32_t* prefix_length,
                                       const int32_t* table, int64_t table_stride, int64_t max_pages, const int32_t* lengths,
                                       float scale, void* o, void* ws, int64_t ws_bytes, void* stream) {
  const CacheGeom kg{kc_sp, kc_sh, kc_ss}, vg{vc_sp, vc_sh, vc_ss};
  TB_CHECK(B >= 0 && H > 0 && H < (int64_t)1 << 24, "paged_attn_prefix: bad shape");
  if (int rc = check_cache("paged_attn_prefix", k_cache, v_cache, pages, Hkv, page, D, kg, vg)) return rc;
  TB_CHECK(H % Hkv == 0, "paged_attn_prefix: query heads must be a multiple of key/value heads");
  TB_CHECK(D <= 256, "paged_attn_prefix: head dim must be at most 256");
  TB_CHECK(max_pages >= 0 && max_pages < (int64_t)1 << 31 && prefix_pages >= 0 && prefix_pages < (int64_t)1 << 31,
           "paged_attn_prefix: table too wide");
  TB_CHECK(aligned16(q) && aligned16(o) && q_sb % 8 == 0 && q_sh % 8 == 0,
           "paged_attn_prefix: q must have 16-byte aligned rows");
  TB_CHECK(aligned4(table) && aligned4(lengths) && aligned4(prefix_table) && aligned4(prefix_length),
           "paged_attn_prefix: tables and lengths must be 4-byte aligned");
  if (B == 0) return 0;
  TB_CHECK(sizes_ok(B, H, Hkv, D), "paged_attn_prefix: shape too large");
  const int64_t top = ((int64_t)1 << 31) - 1024;  // (positions count in 32 bits, tiles past the end included)
  const int64_t pcap = pages == 0 ? 0 : std::min<int64_t>(prefix_pages * page, top);
  // (the plan goes by what the workspace query was asked for, whatever the cache holds)
  const PrefixPlan p = prefix_plan(B, H, Hkv, D, prefix_pages * page, max_pages * page);
  TB_CHECK(B * Hkv * p.own.RG < (int64_t)1 << 31 && Hkv * p.S * p.tiles < (int64_t)1 << 31 &&
               (double)(B * Hkv * p.own.RG) * (double)cdiv(std::min<int64_t>(max_pages * page, (int64_t)1 << 31), kTile) < 2e9,
           "paged_attn_prefix: shape too large");
  TB_CHECK(aligned16(ws) && ws != nullptr, "paged_attn_prefix: workspace missing or misaligned");
  if (ws_bytes < (int64_t)p.bytes) {
    set_error("paged_attn_prefix: workspace too small (%lld bytes, needs %zu)", (long long)ws_bytes, p.bytes);
    return TBF16_EWS;
  }
  uint8_t* const w = (uint8_t*)ws;
  JoinArgs j;
  j.own = attn_args(p.own, q, B, H, Hkv, D, q_sb, q_sh, k_cache, v_cache, pages, page, kg, vg, table, table_stride, max_pages,
                    lengths, scale, o, ws);
  j.own.own = (float*)(w + p.own_part);
  j.own.own_stat = (float*)(w + p.own_stat);
  j.own.where = (int2*)(w + p.where);
  PrefixArgs& a = j.pre;
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.kg = kg;
  a.vg = vg;
  a.table = prefix_table;
  a.length = prefix_length;
  a.cap = (int)pcap;
  a.S = pcap > 0 ? (int)p.S : 0;
  a.pages = (uint32_t)pages;
  a.page = (uint32_t)page;
  a.by_page = div_by(page);
  a.by_group = div_by(H / Hkv);
  a.scale_log2 = j.own.scale_log2;
  a.B = (int)B;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.G = (int)(H / Hkv);
  a.D = (int)D;
  a.part = (float*)(w + p.part);
  a.stat = (float*)(w + p.stat);
  j.keys = p.keys;
  j.unit = p.own.unit;
  j.blocks = (int)p.own.blocks;
  j.o = (uint16_t*)o;
  const hipStream_t st = as_stream(stream);
  if (a.S > 0) {
    launch_prefix(a, p, st);
    TB_LAUNCH_CHECK("paged_attn_prefix");
  }
  launch_attn<true>(j.own, p.own, st);
  TB_LAUNCH_CHECK("paged_attn_prefix own keys");
  prefix_join_kernel<<<(unsigned)cdiv(B * H * (D / 4), 64), kMeet * 64, 0, st>>>(j);
  TB_LAUNCH_CHECK("paged_attn_prefix join");
  return 0;
}
