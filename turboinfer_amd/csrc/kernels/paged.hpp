// paged.hpp -- places of a paged key/value cache and tiles of ragged rows (plain C++: host, device).
#pragma once

#include <stdint.h>

namespace ti {

constexpr int kPagedBlock = 16;               // tokens that share a scale; a page holds whole ones
constexpr float kPagedTiny = 0x1p-100f;       // the least scale

// Block `blk` (tokens 16 blk ..) of a sequence: its number in the cache, [page][kv_head][page / 16], from the table's entry of
// page blk / (page / 16); -1: a hole, or past the table.
struct PagedShape {
  int pages, kv_heads, log_blocks, blocks;    // blocks: of a sequence, table_ld * page / 16
};
constexpr int paged_column(const PagedShape& s, int blk) { return blk >> s.log_blocks; }
constexpr int paged_block(const PagedShape& s, int entry, int head, int blk) {
  if ((unsigned)blk >= (unsigned)s.blocks || (unsigned)entry >= (unsigned)s.pages) return -1;
  return ((entry * s.kv_heads + head) << s.log_blocks) + (blk & ((1 << s.log_blocks) - 1));
}

// Tiles of T rows of ragged sequences without a scan: sequence b's tiles are numbered from paged_tile0(row_start[b], b), so many
// a sequence's rows at most: ceil(n / T) <= floor(n / T) + 1 <= the distance to the next one's.  Numbers between are empty.
constexpr long paged_tile0(long row, int seq, int T) { return row / T + seq; }
constexpr long paged_tiles(long rows, int seqs, int T) { return rows / T + seqs; }   // of all
// The same for 16-token blocks that n rows from any token on touch: <= floor((n + 14) / 16) + 1 <= floor(n / 16) + 2.
constexpr long paged_touch0(long row, int seq) { return row / kPagedBlock + 2 * seq; }
constexpr long paged_touches(long rows, int seqs) { return rows / kPagedBlock + 2 * (long)seqs; }

}  // namespace ti
