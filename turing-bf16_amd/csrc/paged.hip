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
#include "paged_rows.h"

using namespace tbf16;

namespace {

struct CacheGeom {
  int64_t sp, sh, ss;  // element strides of page, head and row
};

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
//
// o = sum_j p_j v_j / sum_j p_j, p_j = exp2(s_j - m), s_j = scale log2(e) q . k_j, with the
// maximum m and both sums running over tiles of 32 keys.
//
// A unit is one sequence's key/value head with up to 16 RT of its query heads (rows). A tile's
// logits are K Q^T on v_mfma_f32_16x16x32_bf16: K rows as they lie in memory (lane l: key l %
// 16, chunks of 8 elements l / 16 + 4 i) against the rows' Q, so lane l gets, for row l % 16,
// keys 4 (l / 16) .. + 3 of each half tile. Those are the lane's 8 k slots of the second
// product O^T = V^T P^T, whose operand P so needs no exchange. V^T's operand holds, for the same
// 8 keys, element dd of chunk l % 16 (chunks of CH = DP / 16): the lane loads its chunk of its
// 8 keys' rows (whole rows per 16 lanes) and picks halves with v_perm_b32, DP / 16 MFMAs per 32
// keys. O^T then has row l % 16's elements CH (4 (l / 16) + i) + dd in lane l: the softmax
// factors of a lane belong to its own outputs. Nothing goes through LDS, every byte of K and V
// is loaded once, by one wave. p goes in as the sum of three bf16, 8 bits of it each: all 24. (Two of
// them lose 2^-17 of p: at 32 sequences of up to 4096 keys the outputs are then 7.4e-5 of their norm off those of
// fp32 products, with three 1.6e-5. They take 0 to 2% less time, 4% with 64 query heads of 64 on a key head.)
//
// Memory bounds it: 16 KB a tile of D = 128 against ~ 550 instructions, 32 of them MFMAs.
// K and V of the next tile are loaded as soon as this tile's registers are free, its page
// entries one tile earlier, across the ends of units too. 128 sequences of 0 to 8192 keys, 8
// heads of 128: 366 us and 5 of the second launch, 5.9 TB/s; a kernel that only reads as many bytes, each
// wave a run of its own: 350 us. 131072 keys of one sequence: 96 and 5 us, 5.6 TB/s (the same reading alone
// 90): ~ 10 us go into the lengths' scan, the first loads, the joins and the second launch. Two tiles a wave
// in registers, blocks of 4 waves or more blocks than run at once were no faster (by 1 to 7%).
//
// Tiles of all units form one list (by sequence, then head). Each wave takes an equal run of
// it, so a batch of ragged lengths keeps every wave busy to the end. What a wave computes of a
// unit that other waves share is joined through LDS inside a block, and through memory and a
// second launch between blocks. Where the cache is so short that a block covers a unit, blocks
// are units and the second launch is left out.

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;
// Running maxima start at kNone; a unit that had any key ends at kFew or above.
constexpr float kNone = -FLT_MAX, kFew = -3.0e38f;
// Weights are at most 1 and go into both sums times kWeight: 256 of the largest values add up without
// overflow. (A maximum that follows only in steps of 2^8, with weights up to 2^8, rescales less often and is
// no faster: 388 and 389 us at 128 sequences, 56 and 57 at 32.)
constexpr float kWeight = 0x1p-8f;

// n / d for 0 <= n < 2^31 as (n magic) >> shift: with d <= 2^l, magic = ceil(2^(31 + l) / d) is off by
// less than 2^-31 of itself.
struct Div {
  uint32_t magic, shift;
};
__device__ __forceinline__ uint32_t operator/(uint32_t n, Div d) { return (uint32_t)((uint64_t)n * d.magic >> d.shift); }

struct AttnArgs {
  const uint16_t *q, *kc, *vc;
  int64_t q_sb, q_sh;
  CacheGeom kg, vg;
  const int32_t *table, *lengths;
  int64_t t_sb;
  int cap;  // positions a table row covers
  uint32_t pages, page;
  Div by_page, by_units, by_blocks, by_waves;  // units of a sequence; blocks and waves of the list form
  float scale_log2;
  int B, H, Hkv, G, D, R, RG;  // R rows a unit, RG units a key/value head
  uint16_t* o;
  float *part, *stat;  // [block][2][R][D], [block][2][R][2]: what a block leaves of units it shares
  int4* desc;  // [block]: the unit it began and later blocks end (b, head, last block, grp + 1), else w = 0
};

__device__ __forceinline__ int seq_len(const AttnArgs& a, int b) { return min(max(a.lengths[b], 0), a.cap); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// A place in the list: tile `tile` of nt of a unit, the grp-th group of R rows of key/value head
// `head` of sequence b.
struct Cursor {
  int b, head, grp, tile, nt, len;
};
__device__ __forceinline__ void advance(const AttnArgs& a, Cursor& c) {
  if (++c.tile < c.nt) return;
  c.tile = 0;
  if (++c.grp < a.RG) return;
  c.grp = 0;
  if (++c.head < a.Hkv) return;
  c.head = 0;
  do {  // (the caller knows that there is a tile ahead)
    if (c.b + 1 >= a.B) c.len = 0;  // unless the lengths change meanwhile: tiles without keys, then
    else c.len = uniform(seq_len(a, ++c.b));
  } while (c.len == 0 && c.b + 1 < a.B);
  c.nt = (c.len + kTile - 1) / kTile;
}
// The list's split: `act` waves of each block (fewer than WPB where the list is so short that the
// CUs would not all get some) take runs of c tiles, run w from tile w c on. This run's length n and
// first place. 32 bits count the list's tiles (the host has made sure).
struct Run {
  uint32_t c, act;
  int n;
  Cursor at;
};
// Inclusive prefix sums over the wave: in rows of 16 lanes, then the rows' last lanes (DPP row_shr 1, 2,
// 4, 8, row_bcast 15 and 31; a scan by ds_bpermute took 0.3 us longer).
__device__ __forceinline__ uint32_t prefix_sum(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
  return v;
}
__device__ __forceinline__ Run run_of(const AttnArgs& a, uint32_t block, uint32_t wave, uint32_t blocks, uint32_t wpb,
                                      int lane) {
  auto length = [&](int b) { return b < a.B ? seq_len(a, b) : 0; };
  auto tiles = [&](int l) { return (uint32_t)((l + kTile - 1) / kTile); };
  auto last = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1); };
  // 64 sequences at a time: a lane's own length and tiles, and those up to its own
  int len = length(lane);
  uint32_t up = prefix_sum(tiles(len)), all = last(up);
  if (a.B > kWave) {
    constexpr int U = 4;
    uint32_t more = 0;
    for (int b = lane + kWave; b < a.B + lane; b += U * kWave) {
      int l[U];
#pragma unroll
      for (int i = 0; i < U; ++i) l[i] = length(b + i * kWave);
#pragma unroll
      for (int i = 0; i < U; ++i) more += tiles(l[i]);
    }
    all += last(prefix_sum(more));
  }
  const uint32_t units = a.Hkv * a.RG;
  all *= units;
  // act = ceil(all / blocks) up to wpb, c = ceil(all / (blocks act))
  Run r{1, wpb, 0, {0, 0, 0, 0, 0, 0}};
  if (all <= blocks * wpb) r.act = max(1u, (all + blocks - 1) / a.by_blocks);
  else r.c = (all + blocks * wpb - 1) / a.by_waves;
  const uint64_t first = ((uint64_t)block * r.act + wave) * r.c;
  if (wave >= r.act || first >= all) return r;
  // the sequence: the first one that ends behind tile `first`
  uint32_t t = (uint32_t)first / a.by_units;  // in tiles of one unit
  const uint32_t rest = (uint32_t)first - t * units;
  int b0 = 0;
  uint64_t past;
  while ((past = __ballot(up > t)) == 0) {
    t -= last(up);
    b0 += kWave;
    if (b0 >= a.B) return r;  // (lengths that changed since they were summed)
    len = length(b0 + lane);
    up = prefix_sum(tiles(len));
  }
  r.n = min(r.c, all - (uint32_t)first);
  const int w = __builtin_ctzll(past);
  r.at.b = b0 + w;
  r.at.len = __builtin_amdgcn_readlane(len, w);
  r.at.nt = (r.at.len + kTile - 1) / kTile;
  t = (t - (__builtin_amdgcn_readlane((int)up, w) - r.at.nt)) * units + rest;  // in the sequence's own tiles
  const uint32_t unit = t / (uint32_t)r.at.nt;
  r.at.tile = t - unit * r.at.nt;
  r.at.head = unit;
  if (a.RG > 1) {
    r.at.head = unit / (uint32_t)a.RG;
    r.at.grp = unit - r.at.head * a.RG;
  }
  return r;
}

// What a lane holds of a unit: for row l % 16 of each 16-row block, the maximum, its own
// part of the sum, and DP / 4 outputs.
template <int DP, int RT>
struct Acc {
  static constexpr int CH = DP / 16;
  float m[RT], l[RT];
  floatx4 o[RT][CH];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      m[r] = kNone;
      l[r] = 0.f;
#pragma unroll
      for (int d = 0; d < CH; ++d) o[r][d] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
  }
  __device__ __forceinline__ void scale(int r, float f) {
    l[r] *= f;
#pragma unroll
    for (int d = 0; d < CH; ++d) o[r][d] *= f;
  }
  // the sum over the four lanes of a row, once, before the unit leaves its wave
  __device__ __forceinline__ void total() {
#pragma unroll
    for (int r = 0; r < RT; ++r) l[r] = sum_xor32(sum_xor16(l[r]));
  }
  // rows of D floats at `rows` (stride ld), their (m, l) at `stat`
  __device__ __forceinline__ void put(float* rows, int ld, float* stat, int R, int D, int lane) const {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = 16 * r + (lane & 15);
      if (row >= R) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < CH; d += 4) {
          const int at = CH * (4 * (lane >> 4) + i) + d;
          if (at < D)
            *reinterpret_cast<float4*>(rows + (int64_t)row * ld + at) =
                make_float4(o[r][d][i], o[r][d + 1][i], o[r][d + 2][i], o[r][d + 3][i]);
        }
      if (lane < 16) *reinterpret_cast<float2*>(stat + 2 * row) = make_float2(m[r], l[r]);
    }
  }
  // adds what n others put, part w at rows + w step and stat + w stat_step: the common maximum
  // first, so that the parts' loads do not wait for each other
  __device__ __forceinline__ void take(const float* rows, int step, int ld, const float* stat, int stat_step, int n, int R,
                                       int D, int lane) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = 16 * r + (lane & 15);
      if (row >= R) continue;
      float mn = m[r];
      for (int w = 0; w < n; ++w) mn = fmaxf(mn, stat[w * stat_step + 2 * row]);
      scale(r, ex2(m[r] - mn));
      m[r] = mn;
#pragma unroll 2
      for (int w = 0; w < n; ++w) {
        const float2 s = *reinterpret_cast<const float2*>(stat + w * stat_step + 2 * row);
        const float f = ex2(s.x - mn);
        l[r] = fmaf(f, s.y, l[r]);
        float4 v[4][CH / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < CH; d += 4)
            v[i][d / 4] = *reinterpret_cast<const float4*>(rows + w * step + row * ld + CH * (4 * (lane >> 4) + i) + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < CH; d += 4) {
            o[r][d][i] = fmaf(f, v[i][d / 4].x, o[r][d][i]);
            o[r][d + 1][i] = fmaf(f, v[i][d / 4].y, o[r][d + 1][i]);
            o[r][d + 2][i] = fmaf(f, v[i][d / 4].z, o[r][d + 2][i]);
            o[r][d + 3][i] = fmaf(f, v[i][d / 4].w, o[r][d + 3][i]);
          }
      }
    }
  }
  // the outputs: o points at the unit's first row
  __device__ __forceinline__ void finish(uint16_t* out, int R, int D, int lane) const {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = 16 * r + (lane & 15);
      if (row >= R) continue;
      const float f = m[r] == kNone ? 0.f : 1.f / l[r];  // no key at all: zeros
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < CH; d += 4) {
          const int at = CH * (4 * (lane >> 4) + i) + d;
          if (at < D)
            *reinterpret_cast<uint2*>(out + (int64_t)row * D + at) =
                make_uint2(pack_bf16(o[r][d][i] * f, o[r][d + 1][i] * f), pack_bf16(o[r][d + 2][i] * f, o[r][d + 3][i] * f));
        }
    }
  }
};

// A unit's first row in o, and how many it has.
__device__ __forceinline__ uint16_t* unit_out(const AttnArgs& a, int b, int head, int grp) {
  return a.o + ((int64_t)b * a.H + head * a.G + grp * a.R) * a.D;
}
__device__ __forceinline__ int unit_rows(const AttnArgs& a, int grp) { return min(a.R, a.G - grp * a.R); }

// DP: D rounded up to 64, 128 or 256 (D == DP unless PAD). WPB waves a block. UNIT: one block
// per unit instead of equal runs of the list.
template <int DP, int RT, int WPB, bool PAD, bool UNIT>
__global__ __launch_bounds__(WPB * 64, DP == 256 ? 1 : DP == 64 && RT == 1 ? 4 : 2) void paged_attn_kernel(AttnArgs a) {
  constexpr int CH = DP / 16, KI = DP / 32, VW = CH / 2;  // V dwords a lane holds of a key
  extern __shared__ __align__(16) float lds[];  // [wave][R][DP + 4], [wave][R][2]
  __shared__ int flags[WPB];  // 1: the wave left a part of a unit begun before it, 2: its last
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r16 = lane & 15;
  constexpr int ld = DP + 4;
  float* const stat0 = lds + WPB * a.R * ld;

  Cursor cur;
  int n;  // this wave's tiles
  int per = 0;  // UNIT: tiles of a wave
  uint32_t c = 0, act = WPB;
  if constexpr (UNIT) {
    cur.b = blockIdx.x;
    cur.head = blockIdx.y;
    cur.grp = blockIdx.z;
    cur.len = uniform(seq_len(a, cur.b));
    cur.nt = (cur.len + kTile - 1) / kTile;
    per = (cur.nt + WPB - 1) / WPB;
    cur.tile = min(wave * per, cur.nt);
    n = min(per, cur.nt - cur.tile);
  } else {
    const Run r = run_of(a, blockIdx.x, wave, gridDim.x, WPB, lane);
    c = r.c;
    act = r.act;
    n = r.n;
    cur = r.at;
    if (threadIdx.x == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (!UNIT && lane == 0) flags[wave] = 0;

  Acc<DP, RT> acc;
  bool tail = false;  // acc is the begin of a unit that goes on in the next wave
  if (n > 0) {
    struct Page {
      int id, row, head;
    };
    // the page and row of the lane's key (l % 32) of a tile
    auto page_of = [&](const Cursor& c) {
      const uint32_t pos = c.tile * kTile + (lane & 31);
      const uint32_t idx = pos / a.by_page;
      Page p{-1, (int)(pos - idx * a.page), c.head};
      if (pos < (uint32_t)c.len) p.id = a.table[c.b * a.t_sb + idx];
      return p;
    };
    uint4 kr[2][KI];
    uint32_t vr[8][VW];
    uint32_t live;  // keys of the tile that there are
    auto shfl_off = [&](int64_t off, int src) {
      return (int64_t)(uint32_t)__shfl((int)off, src, kWave) | (int64_t)__shfl((int)(off >> 32), src, kWave) << 32;
    };
    auto load_k = [&](const Page& p) {
      const bool ok = (uint32_t)p.id < a.pages;
      const int64_t off = ok ? (int64_t)p.id * a.kg.sp + (int64_t)p.row * a.kg.ss : 0;
      const uint16_t* base = a.kc + p.head * a.kg.sh;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint16_t* row = base + shfl_off(off, 16 * h + r16);
#pragma unroll
        for (int i = 0; i < KI; ++i) {
          kr[h][i] = ldg16(row + (PAD ? key_piece(a.D, g, i) : 8 * (g + 4 * i)));
        }
      }
    };
    auto load_v = [&](const Page& p) {
      const bool ok = (uint32_t)p.id < a.pages;
      const int64_t off = ok ? (int64_t)p.id * a.vg.sp + (int64_t)p.row * a.vg.ss : 0;
      auto piece = [&](int i) { return PAD ? value_piece(a.D, DP, r16, i) : CH * r16 + 8 * i; };
      const uint16_t* base = a.vc + p.head * a.vg.sh + piece(0);
      auto load = [&](int j, const uint16_t* at) {
        if constexpr (CH == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(at);
          vr[j][0] = v.x; vr[j][1] = v.y;
        } else {
#pragma unroll
          for (int i = 0; i < value_pieces(DP); ++i) {
            const uint4 v = ldg16(at + (piece(i) - piece(0)));
            vr[j][4 * i] = v.x; vr[j][4 * i + 1] = v.y; vr[j][4 * i + 2] = v.z; vr[j][4 * i + 3] = v.w;
          }
        }
      };
      if ((a.page & 3) == 0) {  // a lane's 4 keys of a half tile lie side by side in one page
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint16_t* at = base + shfl_off(off, 16 * h + 4 * g);
#pragma unroll
          for (int j = 0; j < 4; ++j) load(4 * h + j, at + j * a.vg.ss);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) load(j, base + shfl_off(off, 16 * (j >> 2) + 4 * g + (j & 3)));
      }
    };
    auto alive = [&](const Page& p) { return (uint32_t)__ballot((uint32_t)p.id < a.pages); };  // lanes l and l + 32 alike
    bf16x8 qf[RT][KI];
    auto load_q = [&](const Cursor& c) {
      const int h0 = c.head * a.G + c.grp * a.R, rows = unit_rows(a, c.grp);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int row = 16 * r + r16;
        const uint16_t* src = a.q + c.b * a.q_sb + (h0 + min(row, rows - 1)) * a.q_sh;
#pragma unroll
        for (int i = 0; i < KI; ++i) {
          const int e = 8 * (g + 4 * i);
          const bool in = row < rows && (!PAD || e < a.D);
          const uint4 v = ldg16(src + (!PAD || e < a.D ? e : 0));
          qf[r][i] = __builtin_bit_cast(bf16x8, in ? v : make_uint4(0, 0, 0, 0));
        }
      }
    };

    Page next = page_of(cur);
    load_q(cur);
    load_k(next);
    load_v(next);
    live = alive(next);
    Cursor ahead = cur;
    if (n > 1) {
      advance(a, ahead);
      next = page_of(ahead);
    }
    acc.clear();
    bool begun = cur.tile == 0;  // acc holds its unit from the first tile on
    for (int i = 0;; ++i) {
      const bool more = i + 1 < n;
      Page next2 = next;
      if (i + 2 < n) {
        advance(a, ahead);
        next2 = page_of(ahead);
      }
      // logits
      floatx4 s[RT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          s[r][h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < KI; ++t) {
            uint4 kv = kr[h][t];
            if (PAD && 8 * (g + 4 * t) >= a.D) kv = make_uint4(0, 0, 0, 0);
            s[r][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kv), qf[r][t], s[r][h], 0, 0, 0);
          }
        }
      if (more) load_k(next);
      const bool whole = live == 0xffffffffu;
      bf16x8 pf[RT][3];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = s[r][j >> 2][j & 3] * a.scale_log2;
          if (!whole && !(live >> (16 * (j >> 2) + 4 * g + (j & 3)) & 1)) x[j] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        mx = fmaxf(mx, live ? kFew : kNone);
        mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
        mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
        if (__any(mx > acc.m[r])) {
          const float mn = fmaxf(acc.m[r], mx);
          acc.scale(r, ex2(acc.m[r] - mn));
          acc.m[r] = mn;
        }
        uint32_t f[3][4];  // p's leading 8 bits, the next ones and the last
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float p0 = ex2(x[2 * j] - acc.m[r]) * kWeight, p1 = ex2(x[2 * j + 1] - acc.m[r]) * kWeight;
          acc.l[r] += p0 + p1;
#pragma unroll
          for (int t = 0; t < 3; ++t) {
            f[t][j] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302u);
            p0 -= bf16_hi(__float_as_uint(p0));
            p1 -= bf16_hi(__float_as_uint(p1));
          }
          // 2^-28 of p in place of a part that is zero: an infinite value times it stays infinite
          const ushort2v least = __builtin_elementwise_sub_sat(__builtin_bit_cast(ushort2v, f[0][j]), ushort2v{28 << 7, 28 << 7});
#pragma unroll
          for (int t = 1; t < 3; ++t)
            f[t][j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, f[t][j]), least));
        }
#pragma unroll
        for (int t = 0; t < 3; ++t) pf[r][t] = __builtin_bit_cast(bf16x8, make_uint4(f[t][0], f[t][1], f[t][2], f[t][3]));
      }
      if (!whole) {  // a weight of zero times whatever lies there has to be zero
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(live >> (16 * (j >> 2) + 4 * g + (j & 3)) & 1))
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[j][w] = 0;
      }
#pragma unroll
      for (int d = 0; d < CH; ++d) {
        uint32_t f[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          f[t] = __builtin_amdgcn_perm(vr[2 * t + 1][d >> 1], vr[2 * t][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
        const bf16x8 vf = __builtin_bit_cast(bf16x8, make_uint4(f[0], f[1], f[2], f[3]));
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int t = 0; t < 3; ++t) acc.o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[r][t], acc.o[r][d], 0, 0, 0);
      }
      if (more) {
        load_v(next);
        live = alive(next);
        next = next2;
      }
      const bool end = cur.tile + 1 == cur.nt;  // of the unit
      if (more && (UNIT || !end)) {
        ++cur.tile;
        continue;
      }
      acc.total();
      if constexpr (UNIT) {
        acc.put(lds + wave * a.R * ld, ld, stat0 + wave * a.R * 2, unit_rows(a, cur.grp), a.D, lane);
        break;
      }
      const Cursor done = cur;
      if (more) {  // the next unit's q is on its way while this unit leaves
        advance(a, cur);
        load_q(cur);
      }
      if (begun && end) {
        acc.finish(unit_out(a, done.b, done.head, done.grp), unit_rows(a, done.grp), a.D, lane);
      } else if (!begun) {
        acc.put(lds + wave * a.R * ld, ld, stat0 + wave * a.R * 2, unit_rows(a, done.grp), a.D, lane);
        if (lane == 0) flags[wave] = end ? 3 : 1;
      } else {
        tail = true;
      }
      if (!more) break;
      acc.clear();
      begun = true;
    }
  }
  __syncthreads();
  if constexpr (UNIT) {
    // the waves' parts, a thread 4 outputs of a row
    const int rows = unit_rows(a, cur.grp), dg = a.D / 4;
    const int parts = cur.nt ? (cur.nt + per - 1) / per : 0;
    uint16_t* out = unit_out(a, cur.b, cur.head, cur.grp);
    for (int e = threadIdx.x; e < rows * dg; e += WPB * 64) {
      const int row = e / dg, d = (e - row * dg) * 4;
      float2 st[WPB];
      float m = kNone, l = 0.f;
      floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WPB; ++w) {
        st[w] = w < parts ? *reinterpret_cast<const float2*>(stat0 + (w * a.R + row) * 2) : make_float2(kNone, 0.f);
        m = fmaxf(m, st[w].x);
      }
#pragma unroll
      for (int w = 0; w < WPB; ++w)
        if (w < parts) {
          const float f = ex2(st[w].x - m);
          l = fmaf(f, st[w].y, l);
          o += f * *reinterpret_cast<const floatx4*>(lds + (w * a.R + row) * ld + d);
        }
      const float f = m == kNone ? 0.f : 1.f / l;  // no key at all: zeros
      *reinterpret_cast<uint2*>(out + (int64_t)row * a.D + d) = make_uint2(pack_bf16(o[0] * f, o[1] * f), pack_bf16(o[2] * f, o[3] * f));
    }
    return;
  }
  // joins inside the block: a wave that began a unit takes what the waves after it left, the
  // first wave what they left of a unit begun in an earlier block
  const int64_t slot = (int64_t)blockIdx.x * 2;
  int last;  // the last wave before the end of the unit that wave `from` - 1 goes on with, or of the block
  auto span = [&](int from) {
    for (last = from; last < (int)act - 1 && uniform(flags[last]) == 1; ++last) {
    }
    return uniform(flags[last]) == 3;
  };
  auto take = [&](int from) {
    acc.take(lds + from * a.R * ld, a.R * ld, ld, stat0 + from * a.R * 2, a.R * 2, last + 1 - from, a.R, a.D, lane);
  };
  if (tail) {
    const bool ended = wave + 1 < (int)act && span(wave + 1);
    if (wave + 1 < (int)act) take(wave + 1);
    if (ended) {
      acc.finish(unit_out(a, cur.b, cur.head, cur.grp), unit_rows(a, cur.grp), a.D, lane);
    } else {
      acc.put(a.part + (slot + 1) * a.R * a.D, a.D, a.stat + (slot + 1) * a.R * 2, a.R, a.D, lane);
      // the unit's last tile: this wave's last one is its tile cur.tile
      const uint32_t end = (blockIdx.x * act + wave) * c + n - 1 - cur.tile + cur.nt - 1;
      if (lane == 0) a.desc[blockIdx.x] = make_int4(cur.b, cur.head, end / (c * act), cur.grp + 1);
    }
  }
  if (wave == 0 && uniform(flags[0]) != 0) {
    acc.clear();
    span(0);
    take(0);
    acc.put(a.part + slot * a.R * a.D, a.D, a.stat + slot * a.R * 2, a.R, a.D, lane);
  }
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)  // sequences without keys
    if (uniform(seq_len(a, b)) == 0)
      for (int i = threadIdx.x; i < a.H * a.D / 8; i += WPB * 64)
        stg16(a.o + (int64_t)b * a.H * a.D + 8 * i, make_uint4(0, 0, 0, 0));
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

// How a call is split: head dim DP, RT blocks of 16 rows a unit, wpb waves a block, blocks of
// the list form, and the workspace for what they share.
struct AttnPlan {
  int DP, RT, wpb, R, RG;
  bool unit;  // one block per unit, nothing shared
  int64_t blocks;
  size_t stat, desc, bytes;
};
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

Div div_by(int64_t d) {  // 1 <= d < 2^31
  int l = 0;
  while (((int64_t)1 << l) < d) ++l;
  return Div{(uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d), (uint32_t)(31 + l)};
}

template <int DP, int RT, int WPB>
void launch_attn(const AttnArgs& a, bool unit, int64_t blocks, hipStream_t st) {
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

int check_cache(const char* fn, const void* kc, const void* vc, int64_t pages, int64_t Hkv, int64_t page, int64_t D,
                const CacheGeom& kg, const CacheGeom& vg) {
  TB_CHECK(pages >= 0 && Hkv > 0 && page > 0 && D > 0, "%s: bad cache shape", fn);
  TB_CHECK(pages < (int64_t)1 << 31 && page < (int64_t)1 << 31 && Hkv < (int64_t)1 << 20, "%s: cache too large", fn);
  TB_CHECK(D % 8 == 0, "%s: head dim must be a multiple of 8", fn);
  TB_CHECK(aligned16(kc) && aligned16(vc), "%s: cache must be 16-byte aligned", fn);
  for (const int64_t s : {kg.sp, kg.sh, kg.ss, vg.sp, vg.sh, vg.ss})
    TB_CHECK(s % 8 == 0 && s >= 0 && s < (int64_t)1 << 31, "%s: cache strides must be multiples of 8 below 2^31", fn);
  return 0;
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
  AttnArgs a;
  a.q = (const uint16_t*)q;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.q_sb = q_sb;
  a.q_sh = q_sh;
  a.kg = kg;
  a.vg = vg;
  a.table = table;
  a.lengths = lengths;
  a.t_sb = table_stride;
  a.cap = pages == 0 ? 0 : (int)std::min<int64_t>(max_pages * page, ((int64_t)1 << 31) - 64);
  a.pages = (uint32_t)pages;
  a.page = (uint32_t)page;
  a.by_page = div_by(page);
  a.by_units = div_by(Hkv * p.RG);
  a.by_blocks = div_by(std::max<int64_t>(p.blocks, 1));
  a.by_waves = div_by(std::max<int64_t>(p.blocks * p.wpb, 1));
  a.scale_log2 = scale * 1.4426950408889634f;
  a.B = (int)B;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.G = (int)(H / Hkv);
  a.D = (int)D;
  a.R = p.R;
  a.RG = p.RG;
  a.o = (uint16_t*)o;
  a.part = (float*)ws;
  a.stat = (float*)((uint8_t*)ws + p.stat);
  a.desc = (int4*)((uint8_t*)ws + p.desc);
  const hipStream_t st = as_stream(stream);
#define ATTN(DP_, RT_, WPB_) launch_attn<DP_, RT_, WPB_>(a, p.unit, p.blocks, st)
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
  TB_LAUNCH_CHECK("paged_attn");
  if (!p.unit) {
    paged_join_kernel<<<dim3((unsigned)p.blocks, (unsigned)cdiv(p.R * D, 256)), kJoinWaves * 64, 0, st>>>(a);
    TB_LAUNCH_CHECK("paged_attn join");
  }
  return 0;
}
