// Attention of one new token per sequence over a paged cache where all sequences begin with the same
// tokens: the prefix's keys and values are read once for the whole batch.
//
// o = softmax of the logits of prefix keys and own keys together, times their values. Any split of the keys into
// parts gives (m, l, o) with o = sum_j 2^(x_j - m) v_j and l = sum_j 2^(x_j - m), and parts join as
//   m = max m_i,   l = sum l_i 2^(m_i - m),   o = sum o_i 2^(m_i - m).
// Two launches: the prefix and behind it, in blocks of the same launch, the sequences' own keys (prefix_kernel; the
// latter attn_block of paged_attn.h, which leaves sums instead of outputs), and the join of all parts of a row.
// (The prefix's blocks first: in turns with the others they share CUs unevenly, and took 136 us where alone they took 101.)
#include <cmath>
#include <type_traits>

#include "paged_attn.h"

using namespace tbf16;

namespace {

struct PrefixArgs {
  const uint16_t *q, *kc, *vc;
  int64_t q_sb, q_sh;
  CacheGeom kg, vg;
  const int32_t *table, *length;
  int cap, S, tiles;  // positions the table covers; splits of the keys; tiles of a key/value head's rows
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
// step's; they carry 2^-16, so that sums have the room that paged_attn.h's have). It is a whole number, so that the
// constants added to it and the factors between steps are exact; from 2^22 on it follows at once. Logits are rounded
// products and 2^-16 a factor, as in paged_attn.h: a key has the same weight in the prefix and among the own ones however
// large they are (the product, the difference and 2^-16 in one operation: 180 us a call below instead of 184, and from
// logits of 2^27 on weights that are off by their size). Weights go into the second product with all
// their 24 bits, as the sum of three bf16. (Two of them, 8 bits and the next ones rounded to 8, take 151 us where three
// take 180, for 2012 of 524288 outputs rounded other than the exact value instead of 468; fp32 products: 1014.)
//
// Bound by its instructions where the batch is large: 64 keys and 32 rows of D = 128 are 128 MFMAs, ~ 420 vector
// instructions and 32 exponentials a wave, two units that overlap in part. 128 sequences of 32 heads on 8 key heads,
// 32768 keys and none of their own: 144 us a call with two blocks a CU (477 TFLOPS of the two products as defined, 954 with
// the weights' parts), 162 with one, which leaves half of the CU to the own keys' blocks: with up to 1024 of those a
// sequence a call takes 177 us, with two blocks a CU 186. Where it is small, by a chain: length, page ids, keys, products,
// parts (4 sequences of 16 heads on 700 keys: 7.2 us). (Eight waves on 256 rows in one block were as fast, and slower beside
// own keys.)
//
// LDS: chunk c of 16 bytes of row r lies at chunk c ^ f(r) of its row, so that the 16 rows that a read of
// K takes at one chunk lie in all 64 banks, and so do the two chunks of 8 rows that a transposed read takes.
template <int DP>
__device__ __forceinline__ int swz(int row) {
  if constexpr (DP >= 128) return ((row & 7) << 1) | ((row >> 3) & 1);
  else return (((row >> 1) & 3) << 1) | ((row >> 3) & 1);
}

constexpr int kIds = 2048;  // page ids a block holds at a time
// rows of a unit of own keys
constexpr int own_rows(int DP) { return DP == 256 ? 8 : 16; }
// A row's weights refer to a whole number that its logits pass by at most kLag; by nothing beyond kNear, up to where kLag
// can be added to it exactly.
constexpr float kLag = 8.f, kNear = 0x1p22f;

typedef __attribute__((address_space(1))) void global_void;
__device__ __forceinline__ void load16_lds(const void* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((global_void*)from, (lds_void*)to, 16, 0, 0);
}

// 2^(s c - m - 16), at most 2^(kLag - 16): the product is rounded before the difference, as the maximum's is.
__device__ __forceinline__ float weight(float s, float c, float m) {
#pragma clang fp contract(off)
  const float x = s * c;
  return ex2(x - m) * 0x1p-16f;
}

struct LaunchArgs {
  PrefixArgs pre;
  AttnArgs own;
  int pre_blocks, own_blocks;  // the prefix's blocks first, then those of the own keys
  bool unit;                   // own blocks are units
};

template <int DP, int RB, int WR, int WK, int KB, int ST, bool PAD>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void prefix_kernel(LaunchArgs args) {
  const PrefixArgs& a = args.pre;
  constexpr int NW = WR * WK, KS = 32 * KB * WK, CPR = DP / 8, RPI = 64 / CPR;  // chunks of a row, rows of a load
  constexpr int KPW = KS / RPI / NW;                                             // loads of K a wave does for a stage
  constexpr int KBYTES = KS * DP * 2, STAGE = 2 * KBYTES, KI = DP / 32, DB = DP / 16;
  static_assert(NW == 4 && KS % (RPI * NW) == 0 && ST >= 2 && ST <= 4 && (ST - 2) * 2 * KPW < 63, "stage shape");
  __shared__ __align__(1024) uint8_t st0[STAGE], st1[STAGE], st2[ST > 2 ? STAGE : 16], st3[ST > 3 ? STAGE : 16];
  __shared__ int s_ids[kIds];
  __shared__ float2 s_stat[NW][16 * RB];
  __shared__ int s_flags[NW];
  uint8_t* const stages[4] = {st0, st1, st2, st3};
  int block = blockIdx.x;
  if (block >= args.pre_blocks) {  // own keys
    block -= args.pre_blocks;
    const AttnArgs& o = args.own;
    static_assert(3 * own_rows(DP) * (DP + 4) * 4 <= STAGE, "three waves' rows fit a stage");
    auto rows_of = [&](int w) {
      return w < 3 ? reinterpret_cast<float*>(st0) + w * o.R * (DP + 4) : reinterpret_cast<float*>(st1);
    };
    if (args.unit) {
      const int grp = block % o.RG, bh = block / o.RG, b = bh / o.Hkv;
      attn_block<DP, 1, NW, PAD, true, true>(o, rows_of, &s_stat[0][0].x, s_flags, b, 0, bh - b * o.Hkv, grp);
    } else {
      attn_block<DP, 1, NW, PAD, false, true>(o, rows_of, &s_stat[0][0].x, s_flags, block, args.own_blocks, 0, 0);
    }
    return;
  }
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r16 = lane & 15;
  const int wr = wave % WR, kg = wave / WR;
  // (blocks that read the same keys one behind the other, on one XCD where there are 8 heads)
  const int head = block % a.Hkv, rt = block / a.Hkv % a.tiles, split = block / a.Hkv / a.tiles;
  // read once a block: were another stream to write it meanwhile, waves of several lengths would look up page ids that
  // none of them has loaded
  if (threadIdx.x == 0) s_flags[0] = prefix_len(a.length, a.cap);
  __syncthreads();
  const int length = uniform(s_flags[0]);
  const Splits sp = splits_of(length, KS, a.S);
  const int t0 = split * sp.each, tn = min(sp.each, sp.tiles - t0);
  if (tn <= 0) return;

  const float c = fabsf(a.scale_log2);
  bf16x8 qf[RB][KI];
  floatx4 o[RB][DB];
  float m[RB], up[RB], l[RB];  // m: what the weights refer to, a whole number; up: the largest logit it serves
  bool fresh = true;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m[r] = up[r] = kNone;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[r][d] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  const uint16_t *kc = a.kc + head * a.kg.sh, *vc = a.vc + head * a.vg.sh;
  int id0 = 0, last = 0;  // the first page whose id s_ids holds, the last position it covers
  bool named = true;      // all of these ids name pages
  // page id and row of position pos, or of the last one
  auto page_of = [&](int pos, uint32_t& row) {
    const uint32_t at = min(pos, last), idx = at / a.by_page;
    row = at - idx * a.page;
    return (uint32_t)s_ids[(int)idx - id0];
  };
  // (a wave's loads are rows 16 apart and more, or their chunk is another: see swz)
  const int lrow = lane / CPR, lchunk = lane % CPR;
  const uint32_t k_sp = 2 * (uint32_t)a.kg.sp, k_ss = 2 * (uint32_t)a.kg.ss, v_sp = 2 * (uint32_t)a.vg.sp, v_ss = 2 * (uint32_t)a.vg.ss;
  // Rows of keys that are not there are some row that is: `masked` leaves them out.
  auto issue = [&](uint8_t* stage, int tile) {
#pragma unroll
    for (int j = 0; j < KPW; ++j) {
      const int n = wave + NW * j, krow = n * RPI + lrow, chunk = lchunk ^ swz<DP>(krow);
      uint32_t row, id = page_of(tile * KS + krow, row);
      if (!named) id = id < a.pages ? id : 0;
      uint64_t k = (uint64_t)row * k_ss + ((uint64_t)id * k_sp + (uint64_t)(kc + chunk * 8));
      uint64_t v = (uint64_t)row * v_ss + ((uint64_t)id * v_sp + (uint64_t)(vc + chunk * 8));
      if (PAD && chunk * 8 >= a.D) k = v = (uint64_t)&kZeros;
      load16_lds(reinterpret_cast<const void*>(k), stage + n * 1024);
      load16_lds(reinterpret_cast<const void*>(v), stage + KBYTES + n * 1024);
    }
  };

  // the lane's place in fragments: K row r16, chunk g (+ 4 t); V^T keys 4 g + r16 / 4, columns 4 (r16 % 4)
  const int klane = (kg * 32 * KB + r16) * DP * 2 + ((g ^ swz<DP>(r16)) << 4);
  const int vrow = 4 * g + (r16 >> 2);
  const int vlane = KBYTES + (kg * 32 * KB + vrow) * DP * 2 + (((r16 & 3) >> 1 ^ swz<DP>(vrow)) << 4) + 8 * (r16 & 1);
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4s lds_v4s;

  typedef floatx4 Logits[2][RB];
  typedef bf16x8 Weights[RB][3];
  // 32 keys at a time: logits, ...
  auto logits = [&](const uint8_t* stage, int kl, int h, Logits& s) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < RB; ++r) s[k][r] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KI; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bf16x8 kf = *reinterpret_cast<const bf16x8*>(stage + (kl ^ (t << 6)) + (2 * h + k) * 16 * DP * 2);
#pragma unroll
        for (int r = 0; r < RB; ++r) s[k][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[r][t], s[k][r], 0, 0, 0);
      }
  };
  // ... what the weights refer to, ...
  auto follow = [&](const Logits& s, float cc) {
    float mx[RB];
    bool grown = fresh;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      mx[r] = fmaxf(fmaxf(fmaxf(fmaxf(s[0][r][0], s[0][r][1]), fmaxf(s[0][r][2], s[0][r][3])), fmaxf(s[1][r][0], s[1][r][1])),
                    fmaxf(s[1][r][2], s[1][r][3])) * cc;
      grown |= mx[r] > up[r];
    }
    if (__any(grown)) {
      fresh = false;
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float mn = fmaxf(ceilf(mx[r]), kFew);
        mn = fmaxf(mn, __shfl_xor(mn, 16, kWave));
        mn = fmaxf(mn, __shfl_xor(mn, 32, kWave));
        mn = fmaxf(mn, m[r]);
        const float f = ex2(m[r] - mn);
        m[r] = mn;
        up[r] = fabsf(mn) <= kNear ? mn + kLag : mn;
        l[r] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[r][d] *= f;
      }
    }
  };
  // ... weights, ...
  auto weights = [&](const Logits& s, float cc, Weights& pf) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      uint32_t f[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const floatx4& sv = s[j >> 1][r];
        const float p0 = weight(sv[2 * (j & 1)], cc, m[r]), p1 = weight(sv[2 * (j & 1) + 1], cc, m[r]);
        l[r] += p0 + p1;
        weight_parts(p0, p1, f, j);
      }
#pragma unroll
      for (int t = 0; t < 3; ++t) pf[r][t] = __builtin_bit_cast(bf16x8, make_uint4(f[t][0], f[t][1], f[t][2], f[t][3]));
    }
  };
  // ... and outputs; live: the keys that there are
  auto values = [&](const uint8_t* stage, int vl, int h, const Weights& pf, auto all, uint32_t live) {
    uint4 keep;  // the lane's 8 keys of the 32
    if constexpr (!decltype(all)::value) {
      auto two = [&](int k) { return (live >> k & 1 ? 0xffffu : 0u) | (live >> (k + 1) & 1 ? 0xffff0000u : 0u); };
      keep = make_uint4(two(4 * g), two(4 * g + 2), two(16 + 4 * g), two(18 + 4 * g));
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const uint8_t* at = stage + (vl ^ (d << 5)) + h * 32 * DP * 2;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 16 * DP * 2));
      uint4 v = __builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      // (a weight of zero times whatever lies there has to be zero)
      if constexpr (!decltype(all)::value) v = make_uint4(v.x & keep.x, v.y & keep.y, v.z & keep.z, v.w & keep.w);
      const bf16x8 vf = __builtin_bit_cast(bf16x8, v);
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int t = 0; t < 3; ++t) o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[r][t], o[r][d], 0, 0, 0);
    }
  };
  // A whole tile, from a stage that the next loads must not go into yet. (They go out behind the first reads: where
  // the compiler cannot tell the stages apart it waits for all loads before a read, which by then are those of
  // earlier steps.)
  auto whole = [&](const uint8_t* stage, uint8_t* next, int next_tile) {
    // (opaque, or every stage's addresses are kept in registers of their own)
    int kl = klane, vl = vlane;
    asm volatile("" : "+v"(kl), "+v"(vl));
    Logits s[2];
    Weights pf;
    logits(stage, kl, 0, s[0]);
    issue(next, next_tile);
    follow(s[0], c);
#pragma unroll
    for (int h = 0; h < KB; ++h) {
      if (h + 1 < KB) logits(stage, kl, h + 1, s[(h + 1) & 1]);
      weights(s[h & 1], c, pf);
      values(stage, vl, h, pf, std::true_type(), 0u);
      if (h + 1 < KB) follow(s[(h + 1) & 1], c);
    }
  };
  auto masked = [&](const uint8_t* stage, int tile) {
    for (int h = 0; h < KB; ++h) {
      const int pos = tile * KS + (kg * KB + h) * 32 + (lane & 31);
      uint32_t row;
      const bool there = page_of(pos, row) < a.pages && pos <= last;
      const uint32_t live = (uint32_t)__ballot(there);
      if (live == 0) continue;
      Logits s;
      Weights pf;
      logits(stage, klane, h, s);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[k][r][i] = live >> (16 * k + 4 * g + i) & 1 ? s[k][r][i] * c : -INFINITY;
      follow(s, 1.f);
      weights(s, 1.f, pf);
      values(stage, vlane, h, pf, std::false_type(), live);
    }
  };

  // as many tiles at a time as s_ids covers: the ids, the first loads
  const int most = (int)min((int64_t)tn, max((int64_t)1, (int64_t)(kIds - 2) * a.page / KS));
  auto begin = [&](int done) {
    const int from = (t0 + done) * KS;
    last = min(from + min(most, tn - done) * KS, length) - 1;
    id0 = (int)((uint32_t)from / a.by_page);
    const int ids = (int)((uint32_t)last / a.by_page) - id0 + 1;
    int bad = 0;
    for (int i = threadIdx.x; i < ids; i += NW * 64) {
      const int id = a.table[id0 + i];
      s_ids[i] = id;
      bad |= (uint32_t)id >= a.pages;
    }
    named = __syncthreads_or(bad) == 0;
    // (tiles past the last one load its last row: as many loads in every step, so that it is known without a
    // branch which have come)
#pragma unroll
    for (int u = 0; u < ST - 1; ++u) issue(stages[u], t0 + done + u);
  };
  begin(0);
  // the wave's rows
  const int rows = a.B * a.G, row0 = (rt * WR + wr) * 16 * RB;
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a maximum is looked for: the sign goes to q)
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

  for (int done = 0; done < tn; done += most) {
    const int first = t0 + done, n = min(most, tn - done);
    const int full = named ? (last + 1 - first * KS) / KS : 0;  // whole tiles, in the ring; a last one, or all, on their own
    for (int i0 = 0; i0 < full; i0 += ST) {
#pragma unroll
      for (int u = 0; u < ST; ++u) {
        if (i0 + u >= full) break;
        wait_vmem_n<(ST - 2) * 2 * KPW>();  // stage u is there once only the later stages' loads are on their way
        wait_lds();
        barrier_no_fence();
        whole(stages[u], stages[(u + ST - 1) % ST], first + i0 + u + ST - 1);
      }
    }
    for (int i = full; i < n; ++i) {
      const int u = named ? i % ST : 0;
      if (!named) {
        wait_vmem_n<0>();
        __syncthreads();
        issue(st0, first + i);
      }
      wait_vmem_n<0>();
      __syncthreads();
      masked(u == 0 ? st0 : u == 1 ? st1 : u == 2 ? st2 : st3, first + i);
    }
    if (done + most < tn) {
      wait_vmem_n<0>();
      __syncthreads();  // nobody reads the ids or stages any more, or loads into them
      begin(done + most);
    }
  }
  wait_vmem_n<0>();

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
    // In the terms of paged_attn.h, whose weights are 2^(x - m - 8): the other 2^-8 go to m where that is exact, else to
    // the sums, whose weights are none above 2^-16 then.
    const bool near = fabsf(m[r]) <= kNear;
    const float f = near ? 1.f : 0x1p8f;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const int at = 16 * d + 4 * g;
      if (!PAD || at < a.D) *reinterpret_cast<floatx4*>(a.part + out[r] * a.D + at) = o[r][d] * f;
    }
    if (g == 0) *reinterpret_cast<float2*>(a.stat + out[r] * 2) = make_float2(near ? m[r] + kLag : m[r], l[r] * f);
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

// 64 groups of 4 outputs a block; its waves take a row's parts in turns and meet in LDS. A call with two, four and eight
// waves: 4 sequences of 16 heads on 700 keys 10.7, 10.0, 10.6 us; 13 of 20 heads of 80 on 2999: 15.6, 14.9, 14.7;
// where many rows have few parts (256 of 32 heads on 2048 keys) 61.8, 65.2, 70.4.
constexpr int kMeet = 4;
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

// How a call is split: rows of a block and keys of a tile by the form, splits of the prefix, own keys.
struct PrefixPlan {
  int DP, few, rows, keys;
  int64_t tiles, S;  // row tiles of a key/value head, splits
  AttnPlan own;
  size_t part, stat, own_part, own_stat, where, bytes;
};
PrefixPlan prefix_plan(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t prefix_cap, int64_t cap) {
  PrefixPlan p;
  const int64_t G = H / Hkv, n = B * G;
  p.DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  p.keys = p.DP == 256 ? 32 : 64;
  const int64_t all = cdiv(prefix_cap, p.keys);
  // Blocks of 64 rows, two groups of waves on different keys, or of 128, which read the keys half as often: the former
  // where a CU would get up to 8 tiles of the latter, or the rows leave a fifth and more of 128 empty (8 heads, 64 and 128:
  // 128 rows on 4096 keys 21.9 and 25.5 us, 256 rows 26.2 and 26.7, 512 rows 36.1 and 36.0, 256 rows on 32768 keys 96.9 and
  // 90.1, 160 rows 80.6 and 88.2; one head, 256 rows on 4096: 15.9 and 19.1. Against it: 4 heads of 80, 65 rows on 2999
  // keys: 15.5 and 14.9; of 64, 800 rows on 512: 15.0 and 14.1).
  p.few = p.DP < 256 && ((double)(Hkv * cdiv(n, 128)) * (double)all <= 8.0 * (double)num_cus() ||
                         5 * cdiv(n, 128) * 128 >= 6 * cdiv(n, 64) * 64);
  p.rows = p.DP == 256 || p.few ? 64 : 128;
  p.tiles = cdiv(n, p.rows);
  // Splits: a block a CU, which leaves half of its room to the own keys' blocks (256 rows of 8 heads on 8192 keys
  // and up to 512 own ones a sequence: 37.1 us, two blocks a CU 45.2; without own ones 34.2 and 32.5), but no more than
  // pays for the parts they leave: a tile takes a block ~ 1.3 us, a split's part of all rows 8 bytes an element at 8 TB/s and
  // 0.05 us of the join (65 rows of 4 heads of 80 on 2999 keys: 15.5 us, with up to twice as many splits 15.9).
  const double part_us = (double)(B * H * D) * 1e-6 + 0.05;
  const int64_t most = std::max<int64_t>(1, (int64_t)std::sqrt(1.3 * (double)all / part_us));
  p.S = std::min({all, most, std::max<int64_t>(1, num_cus() / (Hkv * p.tiles))});

  AttnPlan& o = p.own;
  o.DP = p.DP;
  o.RT = 1;
  o.wpb = 4;
  o.R = (int)std::min<int64_t>(G, own_rows(p.DP));
  o.RG = (int)cdiv(G, o.R);
  // (a block a unit as long as that is a few tiles a wave: 32 sequences of up to 512 keys, 8 heads, behind 4096:
  // 22.2 us, as a list 27.7; 64 behind 8192: 37.1 and 38.0; very many short units are joined to runs)
  o.unit = cdiv(cap, kTile) <= 4 * o.wpb && B * Hkv * o.RG <= 4 * num_cus();
  o.blocks = o.unit ? B * Hkv * o.RG : 2 * num_cus();
  o.stat = align_up((size_t)o.blocks * 2 * o.R * (size_t)D * 4, 256);
  o.desc = o.bytes = o.unit ? 0 : o.stat + align_up((size_t)o.blocks * 2 * o.R * 2 * 4, 256);
  p.part = o.bytes;
  p.stat = p.part + align_up((size_t)(p.S * B * H * D) * 4, 256);
  p.own_part = p.stat + align_up((size_t)(p.S * B * H) * 8, 256);
  p.own_stat = p.own_part + align_up((size_t)(B * H * D) * 4, 256);
  p.where = p.own_stat + align_up((size_t)(B * H) * 8, 256);
  p.bytes = p.where + align_up((size_t)(B * Hkv * o.RG) * 8, 256);
  return p;
}

template <int DP, int RB, int WR, int WK, int KB, int ST>
void launch_form(const LaunchArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)(a.pre_blocks + a.own_blocks);
  if (a.pre.D == DP) prefix_kernel<DP, RB, WR, WK, KB, ST, false><<<grid, 256, 0, st>>>(a);
  else prefix_kernel<DP, RB, WR, WK, KB, ST, true><<<grid, 256, 0, st>>>(a);
}
void launch_prefix(const LaunchArgs& a, const PrefixPlan& p, hipStream_t st) {
  if (p.DP == 64) {
    if (p.few) launch_form<64, 2, 2, 2, 1, 4>(a, st);
    else launch_form<64, 2, 4, 1, 2, 4>(a, st);
  } else if (p.DP == 128) {
    if (p.few) launch_form<128, 2, 2, 2, 1, 2>(a, st);
    else launch_form<128, 2, 4, 1, 2, 2>(a, st);
  } else {
    launch_form<256, 1, 4, 1, 1, 2>(a, st);
  }
}

bool sizes_ok(int64_t B, int64_t H, int64_t Hkv, int64_t D) {
  // (the join: 256 threads for 64 groups of 4 outputs, below 2^32 in all)
  return B > 0 && H > 0 && Hkv > 0 && D > 0 && D <= 256 && H % Hkv == 0 && H < (int64_t)1 << 24 &&
         (double)B * (double)H < 1e9 && (double)(B * H) * (double)(D / 4) <= 1073741824.0 - 64.0;
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
  TB_CHECK(B * Hkv * p.own.RG < (int64_t)1 << 31 && Hkv * p.S * p.tiles + p.own.blocks < (int64_t)1 << 31 &&
               (double)(B * Hkv * p.own.RG) * (double)cdiv(std::min<int64_t>(max_pages * page, (int64_t)1 << 31), kTile) < 2e9,
           "paged_attn_prefix: shape too large");
  TB_CHECK(aligned16(ws) && ws != nullptr, "paged_attn_prefix: workspace missing or misaligned");
  if (ws_bytes < (int64_t)p.bytes) {
    set_error("paged_attn_prefix: workspace too small (%lld bytes, needs %zu)", (long long)ws_bytes, p.bytes);
    return TBF16_EWS;
  }
  uint8_t* const w = (uint8_t*)ws;
  LaunchArgs la;
  la.own = attn_args(p.own, q, B, H, Hkv, D, q_sb, q_sh, k_cache, v_cache, pages, page, kg, vg, table, table_stride, max_pages,
                     lengths, scale, o, ws);
  la.own.own = (float*)(w + p.own_part);
  la.own.own_stat = (float*)(w + p.own_stat);
  la.own.where = (int2*)(w + p.where);
  la.unit = p.own.unit;
  PrefixArgs& a = la.pre;
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
  a.tiles = (int)p.tiles;
  a.pages = (uint32_t)pages;
  a.page = (uint32_t)page;
  a.by_page = div_by(page);
  a.by_group = div_by(H / Hkv);
  a.scale_log2 = la.own.scale_log2;
  a.B = (int)B;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.G = (int)(H / Hkv);
  a.D = (int)D;
  a.part = (float*)(w + p.part);
  a.stat = (float*)(w + p.stat);
  la.pre_blocks = (int)(Hkv * a.S * p.tiles);
  la.own_blocks = (int)p.own.blocks;
  JoinArgs j{la.own, la.pre, p.keys, p.own.unit, (int)p.own.blocks, (uint16_t*)o};
  const hipStream_t st = as_stream(stream);
  launch_prefix(la, p, st);
  TB_LAUNCH_CHECK("paged_attn_prefix");
  prefix_join_kernel<<<(unsigned)cdiv(B * H * (D / 4), 64), kMeet * 64, 0, st>>>(j);
  TB_LAUNCH_CHECK("paged_attn_prefix join");
  return 0;
}
