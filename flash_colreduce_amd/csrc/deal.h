// How the work of tree_attention is cut, in whole numbers: the kernels', the join's and the host's side of it.  Plain C++, so that it can be
// tested without a device.
//
// An item is 16 rows and more of a (sequence, head) and all of its keys, in blocks of kBlock.  Blocks of all items are laid end to end and every workgroup
// takes `per` of them, or (most_of) items are cut into pieces of one item each, a workgroup for each.  Of an item that was cut the workgroup with its first part
// tells the join how many blocks others have; from that the join knows how many workgroups these are (followers), one behind the other.
#pragma once

#include "div.h"

namespace fcr_tree {

constexpr int kBlock = 128;                  // keys of a block

FCR_HOST_DEVICE inline int least_of(int a, int b) { return a < b ? a : b; }
FCR_HOST_DEVICE inline int quotient_up(int a, int b) { return (int)((uint32_t)(a + b - 1) / (uint32_t)b); }

FCR_HOST_DEVICE inline int blocks_of(int n) { return n <= 0 ? 1 : (n + kBlock - 1) / kBlock; }

// Pieces of one item each, where some number of blocks a little above `per` makes them no more than the workgroups.  A
// second piece costs a workgroup of many rows as much as 2.6 blocks (first stage, partial results, code that runs for the first time), and row
// tiles whose pieces are cut alike read the same keys at the same time.  256 rows over 4 x 8 heads of 8192 keys of 128 elements: 77 -> 73 us bf16,
// 79 -> 74 int8; 32 rows: 53 -> 35 bf16, 36 -> 34 int8; 40 rows over 3 x 7 heads of 30000 keys bf16 139 -> 97.  Few rows of one tile
// (8 x 8 heads of 8192 keys, one token: 55 -> 50 bf16, 36 -> 33 int8) lose 0.7 us where there is none, too much for less than 8 blocks.
FCR_HOST_DEVICE inline bool pieces_are_tried(int entries, int threads, int per, int row_tiles, bool tall) {
  return entries <= threads && (tall || row_tiles > 1 || per >= 8);
}
FCR_HOST_DEVICE inline int most_allowed(int per, int row_tiles, bool tall) {
  return per + (tall ? 2 : 0) + least_of(per / 8, row_tiles > 1 ? 6 : tall ? 0 : 2);
}
// The least number of blocks from `per` to `limit` that fits, 0 if there is none; fits(it) was called last.  More blocks never make more pieces, so
// that `limit` tells whether there is one.
template <class Fits>
FCR_HOST_DEVICE inline int most_of(int per, int limit, Fits fits) {
  int p = limit;
  for (bool found = false;;) {
    const bool fit = fits(p);
    if (!found && !fit) return 0;
    if (fit && (found || p == per)) return p;
    p = found ? p + 1 : per;                 // (`limit` again at most)
    found = true;
  }
}
// An item's pieces, and the blocks of all but its last one (which has one at least).
FCR_HOST_DEVICE inline int pieces_of(int blocks, int most) { return quotient_up(blocks, most); }
FCR_HOST_DEVICE inline int piece_length(int blocks, int pieces) { return quotient_up(blocks, pieces); }

// Workgroups behind the one with an item's first part that have parts of it: `others` blocks are theirs.  unit: `per`, or the pieces' `most`.
FCR_HOST_DEVICE inline int followers(int others, int unit) { return others <= 0 ? 0 : quotient_up(others, unit); }

// Which kernel takes `rows` rows of a (sequence, head) of at most 64 w elements: 1, tree_attention_kernel; 4 and 8, tall_attention_kernel of as many
// waves (4: of at most 128 elements, see tall_tiles).
// Both sides, us, at 4 sequences x 8 heads x 8192 keys, int8 (bf16): 48 rows of 64 elements 33 (31) by form 1, 37 (33) by form 4, 64 rows 38
// (35) and 38 (34); of 128 elements 42 (45) and 47 (46), 48 (52) and 49 (47); 48 rows of 256 elements 59 (89) by form 1, 62 (61) by form 8, 64
// rows 69 (108) and 65 (67); 128 rows of 128 elements 58 (57) by form 4, 60 (64) by form 8, 192 rows 77 (79) and 72 (74).
FCR_HOST_DEVICE inline int form_of(int64_t rows, int w, bool codes) {
  if (rows <= (w <= 2 || codes ? 48 : 16)) return 1;
  return w <= 2 && rows <= 128 ? 4 : 8;
}
// Column tiles per wave of tall_attention_kernel: two, where their sums and queries leave room in 256 registers.
FCR_HOST_DEVICE constexpr int tall_tiles(int w) { return w <= 2 ? 2 : 1; }
// Rows of an item.
FCR_HOST_DEVICE inline int rows_of_tile(int form, int w) { return form == 1 ? 16 : 16 * tall_tiles(w) * form; }

}  // namespace fcr_tree
