// Where a thread's piece of pages lies. Plain C++ (constexpr, so that kernels have it too): indexes past
// 32 bits are checked without a device.
#pragma once

// Piece `at` of pages of 2^page_shift tokens, PIECES (a power of two) to a token: the row (of pages and
// heads), the token's slot in it and the piece of the token.
struct PagedPiece {
  int row, slot, piece;
};
template <int PIECES>
constexpr PagedPiece paged_piece(long long at, int page_shift) {
  static_assert(PIECES > 0 && (PIECES & (PIECES - 1)) == 0, "");
  const long long token = at / PIECES;
  return {(int)(token >> page_shift), (int)token & ((1 << page_shift) - 1), (int)(at % PIECES)};
}

// Places that blocks of 16 tokens with new ones may take, from request 0's on: the first of request b, whose
// new tokens are rows from `start` on. n tokens lie in at most n / 16 + 2 blocks, and a request of n has so
// many places or more.
constexpr int paged_block_place(int start, int b) { return start / 16 + 2 * b; }

// Elements from the start of a page's head to its slot, 128 each (pages of 2^24 tokens and more pass 32 bits).
constexpr long long paged_slot_at(int slot) { return (long long)slot * 128; }
