// How an 8-bit linear runs: the choice among the kernels of gemm_i8.hip by M, K, N, whether x's rows
// are whole 16-byte chunks (vec) and the device's compute units. Plain C++, so that what a set of
// shapes covers can be asked without a GPU.
#pragma once
#include <algorithm>

#include "sizes.h"

namespace tbf16::i8 {

// The decode kernel's limits: tokens; codes quantised in its blocks (of 2 tokens four times as many),
// values a row of 5 and more.
constexpr int kDecodeRows = 16, kFusedCodes = 16384, kFusedK = 4096;

// The tile kernels (gemm_tiles.h), and the estimate of their times: a round of at most CU-count
// blocks takes c1 + k tiles x slope us, the slope from `light` (few blocks) to `full`, a k tile being
// 128 integers; splitting K over s blocks a tile adds the partial sums' round trip and a launch.
// The figures are those of the fp16 kernels by 128 bytes of k: the MFMAs take as long, and so do
// LDS and L2, which bound both. On 30 shapes (M 16 to 8192) the tile they pick is the best one's time
// but for 1% on average, 7% at most. 4096^3: 52 us, 2640 TOPS, MFMAs busy 0.56 at 2.2 GHz. The direct
// loads' way into LDS beside the MFMAs costs the most of the rest: timed at 4096 x 16384 x 4096, 234 us a
// call, 175 with the loop's loads left out, 230 with all of them from one place (so not HBM), 227 with
// half of x's LDS reads. The weight from memory to registers, only x through LDS, is slower (336 us).
struct Tile {
  int bm, bn;
  bool ksplit;
  float c1, light, full;
};
constexpr Tile kTiles[] = {{256, 256, false, 7.6f, 0.97f, 1.40f}, {192, 256, false, 7.4f, 0.82f, 1.04f},
                           {128, 256, false, 5.8f, 0.75f, 0.87f}, {256, 128, false, 5.8f, 0.66f, 0.87f},
                           {256, 128, true, 6.6f, 0.62f, 0.83f},   {192, 128, true, 5.6f, 0.46f, 0.635f},
                           {128, 128, true, 3.9f, 0.44f, 0.52f},   {128, 64, true, 2.7f, 0.36f, 0.37f},
                           {64, 128, true, 2.7f, 0.36f, 0.37f},    {64, 64, true, 2.0f, 0.25f, 0.26f}};
constexpr int kNumTiles = sizeof(kTiles) / sizeof(kTiles[0]);
constexpr size_t kSplitBytes = (size_t)16 << 20;

// How a call runs.
struct Plan {
  bool decode;        // the decode kernel, else a tile kernel
  int T, R, fused;    // decode: R weight rows a block in T tiles of 16; its FUSED
  int tile, splits;   // tiles: which of kTiles, parts of K
  int rows;           // weight rows a tile takes: fewer than bn where a single row of tiles would leave CUs idle
  size_t scale, x8, part, bytes;  // workspace
};

inline Plan plan_of(int64_t M, int64_t K, int64_t N, bool vec, int64_t cus) {
  Plan p{false, 1, 1, 0, 0, 1, 0, 0, 0, 0, 0};
  const int64_t Kp = (int64_t)align_up((size_t)K, 128), Np = (int64_t)align_up((size_t)N, 8);
  if (M <= kDecodeRows) {
    p.R = (int)std::min<int64_t>(64, std::max<int64_t>(8, cdiv(cdiv(N, cus), 8) * 8));
    p.T = (int)cdiv(p.R, 16);
    p.decode = true;
    if (vec && (M * Kp <= (M <= 2 ? 4 : 1) * kFusedCodes || Kp <= kFusedK)) {
      p.fused = M == 1 ? 1 : M <= 4 ? 2 : 3;
      return p;
    }
  }
  p.x8 = align_up((size_t)M * 4, 256);
  p.bytes = p.part = align_up(p.x8 + (size_t)M * Kp, 256);
  if (p.decode) return p;
  const int64_t KT = std::max<int64_t>(1, Kp / 128);
  float best = 1e30f;
  for (int i = 0; i < kNumTiles; ++i) {
    const Tile& t = kTiles[i];
    const int64_t tiles = cdiv(M, t.bm) * cdiv(N, t.bn);
    if (tiles >= (int64_t)1 << 31) continue;
    for (int s = 1; s <= 8; s *= 2) {
      const int64_t kt = cdiv(KT, s);
      if (s > 1 && (kt < 8 || (s - 1) * kt >= KT || (size_t)s * M * Np * 4 > kSplitBytes)) break;
      const float load = std::min(1.f, (float)(tiles * s) / (float)cus);
      float us = (float)cdiv(tiles * s, cus) * (t.c1 + (float)kt * (t.light + (t.full - t.light) * load));
      if (s > 1) us += 4.5f + (float)s * (float)M * (float)Np * 8.f / 2e6f;
      if (us < best) {
        best = us;
        p.tile = i;
        p.splits = s;
      }
    }
  }
  const Tile& t = kTiles[p.tile];
  p.rows = t.bn;
  if (t.ksplit && M <= t.bm && p.splits == 1 && cdiv(N, t.bn) < cus)
    p.rows = (int)std::min<int64_t>(t.bn, std::max<int64_t>(8, cdiv(cdiv(N, cus), 8) * 8));
  if (p.splits > 1) p.bytes = p.part + (size_t)p.splits * M * Np * 4;
  return p;
}

}  // namespace tbf16::i8
