// Which elements of a key's or value's row of D elements the lanes of the paged attention load:
// plain C++, so that every D can be checked without a GPU. D % 8 == 0, DP is D rounded up to 64,
// 128 or 256. What a lane loads in place of elements past D goes to products or outputs that are
// left out; the address has to lie in the row all the same, the last row of a cache may end its
// memory.
#pragma once

namespace tbf16 {

// Element e, or the row's first where there is no e.
constexpr int in_row(int D, int e) { return e < D ? e : 0; }

// K: 8 elements at a time, piece i of lane group g (lane / 16).
constexpr int kKeyPiece = 8;
constexpr int key_pieces(int DP) { return DP / 32; }
constexpr int key_piece(int D, int g, int i) { return in_row(D, 8 * (g + 4 * i)); }

// V: a chunk of DP / 16 elements of lane r16 (lane % 16), in pieces of at most 8 (DP = 256: two, of
// which the row may hold the first alone).
constexpr int value_piece_size(int DP) { return DP == 64 ? 4 : 8; }
constexpr int value_pieces(int DP) { return DP / 16 / value_piece_size(DP); }
constexpr int value_piece(int D, int DP, int r16, int i) { return in_row(D, DP / 16 * r16 + 8 * i); }

// No lane's loads leave a row, for any D that DP serves.
constexpr bool rows_kept(int DP) {
  for (int D = DP == 64 ? 8 : DP / 2 + 8; D <= DP; D += 8) {
    for (int g = 0; g < 4; ++g)
      for (int i = 0; i < key_pieces(DP); ++i)
        if (key_piece(D, g, i) + kKeyPiece > D) return false;
    for (int r = 0; r < 16; ++r)
      for (int i = 0; i < value_pieces(DP); ++i)
        if (value_piece(D, DP, r, i) + value_piece_size(DP) > D) return false;
  }
  return true;
}
static_assert(rows_kept(64) && rows_kept(128) && rows_kept(256), "a lane reads past its row");

}  // namespace tbf16
