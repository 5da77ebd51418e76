// How the work of tree_attention and chunk_attention is cut, in whole numbers: the kernels', the join's and the host's side of it.  Plain C++, so that it can be
// tested without a device.  Sight, Steps and what stands behind them are chunk_attention's alone.
//
// An item is 16 rows and more of a (sequence, head) and all of its keys, in blocks of kBlock.  Blocks of all items are laid end to end and every workgroup
// takes `per` of them, or (most_of) items are cut into pieces of one item each, a workgroup for each.  Of an item that was cut the workgroup with its first part
// tells the join how many blocks others have; from that the join knows how many workgroups these are (followers), one behind the other.
#pragma once

#include <stdint.h>

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

// Which kernel takes `rows` rows of a (sequence, head) of at most 64 w elements: 1, few_attention_kernel; 4 and 8, tall_attention_kernel (chunk_attention:
// chunk_attention_kernel) of as many waves (4: of at most 128 elements, see tall_tiles).
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

FCR_HOST_DEVICE inline int most_of_two(int a, int b) { return a > b ? a : b; }

// What tokens first .. last of a sequence (those that it has) see in chunk_attention: keys of [lo, n) and [0, prefix), and no others; keys of [all_lo, all_hi) and
// [0, prefix), every token.  Blocks that begin at gap_at or behind it (a number of keys) lie `gap` keys further back than their number says: between the
// prefix and lo no key is seen.  They are taken from the last one to the first: where scores lose a slope times the distance the largest weights come first, and
// the reference of a row rises once, not with every step towards the token (two prompts of up to 4096 biased tokens, 16 heads: 306 -> 240 us).  (context
// up to 2^30, T up to 2^24.)
constexpr int kNoKey = 0x7fff0000;           // above every n
struct Sight {
  int context, n, lo, all_lo, all_hi, prefix, gap_at, gap;
  FCR_HOST_DEVICE Sight() {}
  FCR_HOST_DEVICE Sight(int context_, int count, int prefix_, int window, int T, int positions, int first, int last) {
    context = least_of(most_of_two(context_, 0), 1 << 30);
    count = least_of(most_of_two(count, 0), T);
    last = least_of(last, count - 1);
    const bool none = first >= count;
    const int there = least_of(context + count, positions);
    prefix = none ? 0 : least_of(most_of_two(prefix_, 0), there);
    n = none ? 0 : least_of(there, most_of_two(context + last + 1, prefix));
    lo = least_of(most_of_two(context + first + 1 - window, 0), n);
    all_lo = most_of_two(context + last + 1 - window, 0);
    all_hi = least_of(context + first + 1, n);
    gap_at = (prefix + kBlock - 1) & -kBlock;
    gap = most_of_two((lo & -kBlock) - gap_at, 0);
  }
  FCR_HOST_DEVICE int blocks() const { return most_of_two((n - gap + kBlock - 1) / kBlock, 1); }
  // The key at x of the blocks laid end to end; kNoKey in front of them.
  FCR_HOST_DEVICE int key(int x) const { return x < 0 ? kNoKey : x + (x >= gap_at ? gap : 0); }
  // The key that lies `at` keys behind the first one of the blocks where the last block is in front.
  FCR_HOST_DEVICE int position(int at) const {
    const int from = ((n - gap + kBlock - 1) & -kBlock) - kBlock - (at & -kBlock);
    return from < 0 || at < 0 ? kNoKey : key((at & (kBlock - 1)) + from);
  }
  // whether every token sees `len` keys from pos on
  FCR_HOST_DEVICE bool whole(int pos, int len) const { return (pos >= all_lo && pos + len <= all_hi) || pos + len <= prefix; }
  FCR_HOST_DEVICE bool settled(int pos, int len) const { return whole(pos, len); }
};

// What some rows of an item see of the item's steps of 32 keys, a step named by its first key's x.
struct Steps {
  int fast, fasts, high, low, prefix;
  FCR_HOST_DEVICE Steps(const Sight& rows, const Sight& item, bool live) {
    fast = rows.all_lo - item.gap;
    fasts = most_of_two(rows.all_hi - 31 - rows.all_lo, 0);
    high = !live ? 0 : rows.n > item.gap_at ? rows.n - item.gap : rows.n;
    low = rows.lo - item.gap - 32;
    prefix = live ? rows.prefix : 0;
  }
  // some row might see one of the keys; every row sees all of them
  FCR_HOST_DEVICE bool some(int x) const { return x < prefix || (x < high && x > low); }
  FCR_HOST_DEVICE bool whole(int x) const { return (uint32_t)(x - fast) < (uint32_t)fasts || x <= prefix - 32; }
  // of all steps from `first` down to `last`
  FCR_HOST_DEVICE bool whole(int first, int last) const { return (last >= fast && first - fast < fasts) || first <= prefix - 32; }
};

// Blocks that an item of chunk_attention has at most; window: 0 where there is none, or a prefix, whose length only the device knows.
FCR_HOST_DEVICE inline int64_t most_blocks_of(int64_t positions, int window, int tile_rows, int G) {
  const int64_t near = (int64_t)window + tile_rows / G + 2 * kBlock;
  return ((window && near < positions ? near : positions) + kBlock - 1) / kBlock;
}
// few_attention_kernel takes more rows than form_of gives it, in tiles of 16, where the chip has few of them: it starts faster and its items are many, so that they run at once and
// need not be cut.  us, by it and by the kernel for many rows, at the largest size on its side and the next one: 8 x 8 fp16 heads of 128 rows of 128 elements, 1564 keys 36.0, 41.6,
// 256 rows, 464 keys 26.5, 31.9, 1564 keys 63.4, 49.4; of 64 elements 256 rows, 464 keys 16.7, 22.0, 1564 keys 39.2, 35.4; of 256 elements 128 rows, 464 keys 32.5, 39.9, 1564 keys
// 72.0, 57.7; e4m3 keys of 128 elements, 512 rows, 178 keys 24.9, 25.7, 528 keys 40.7, 38.4.  One item of 64 rows of 128 elements and 114 keys: 7.5, 16.0.
FCR_HOST_DEVICE inline bool takes_few_rows(int64_t items, int held, int64_t longest) { return items * (longest + 2) <= 15ll * held; }
// Tiles of 128 rows, two workgroups to a CU, instead of 256, where there are more than the chip holds and they are short or mostly of keys that only some of the rows see: less is
// multiplied that is hidden, and what runs once for one tile runs beside the other one's products.  fp16, us, 128 rows and 256: 64 elements, 128 prompts of 384 tokens, 16 heads, 159, 230;
// 8 of 2048 of 8 heads of 4 queries 261, 272, 2 of 4096 of 16 heads 148, 141; 64 chunks of 64 behind 300 keys 42, 44, 16 of 512 behind 2000 265, 267; 128 elements: 16 of 768
// 196, 206, 8 of 1024 152, 145, 32 of 256 behind 500 keys 184, 181.
FCR_HOST_DEVICE inline bool takes_half_tiles(int64_t items, int held, int64_t longest, int D, int64_t positions, int T) {
  return items > held && (positions <= 2ll * T ? longest <= (D <= 64 ? 16 : 6) : D <= 64 && longest <= 6);
}

// Items of chunk_attention may be taken whole, a workgroup for each, by a launch of as many: nothing is cut and joined, tiles of one head run together on one die, but the last
// workgroups may leave others idle.  2: they are, without a look at the lengths or the launch that joins, where the longest that there can be (blocks of it) is no more
// than some for each that a workgroup gets: keys of tall tiles (many rows) are bound by the matrix instructions wherever they are, few rows by memory, of which
// the last workgroups have the more.  1: if items_are_whole says so.  0: no.
//   One token of 8 heads of fp16 keys of 128 elements, us, cut and whole: 450 keys 10.9, 9.2; 900 11.3, 13.5; of 16 sequences 18.9, 16.3; 2000 of 64, of drawn lengths 64, 55.
//   Many rows: 4 chunks of 512 tokens, 8 heads of 4 queries, behind 1000 keys 104, 73; 16 of 300 tokens of 256 elements 247, 215.
FCR_HOST_DEVICE inline int whole_items_of(int64_t items, int held, int64_t longest, bool tall) {
  if (longest * held <= (tall ? 2 * held + 12 * items : 4 * held + 16 * items)) return 2;
  return (tall ? 4 * items : items) >= held ? 1 : 0;
}
// Blocks that what runs once for an item counts as where items are laid end to end: workgroups that have many short ones would take longer than the others.  No more
// than half of a workgroup's blocks, or where there are few a part of them would get nothing else.  16 chunks of 128 tokens behind up to 2000 keys of 128 elements, 8 heads of 4
// queries: 121 us without, 85 with them (five: 91); 64 heads of 8192 tokens 1520 and 1200; one token of 64 sequences of up to 2000 e4m3 keys 52 and 38.
FCR_HOST_DEVICE inline int once_of(int per, bool tall) { return least_of(tall ? 3 : 1, per / 2); }
// Whether items of these weights (blocks and what runs once) are better taken whole.  They take as long as the longest of them or, where there is more than one for
// a workgroup, as their mean and a part of the longest; cut ones as their mean, what runs once for a second piece, and the join.  8 heads of 4096 fp16 tokens, two prompts:
// 131 us cut and 154 whole; 4 chunks of 512 tokens, one behind 8192 keys, the others behind 512: 122 and 277, all behind 8192 370 and 340.
FCR_HOST_DEVICE inline bool items_are_whole(int longest, int per, int items, int held, bool tall) {
  return (items <= held ? longest : most_of_two(longest, per + longest / 8)) <= per + (tall ? 6 : 5);
}

}  // namespace fcr_tree
