// pages4.h -- where a pool of 4-bit pages keeps what (the form is in include/linmt_decoder.h).  Host and device: the tests
// check the same functions on the CPU.
//
// The order inside a tile is the order in which the lanes of a warp hold the right-hand operand of mma.m16n8k16 (lane = 4 g + c
// has column g and rows 2 c, 2 c + 1, 2 c + 8, 2 c + 9), so that the attention kernel loads 16 bytes a lane, lane after lane, and unpacks them
// in place: no shuffle, no bank conflict.  Keys: a column is a position and the rows are components, whose order is free as
// long as the queries follow it.  Values: a column is a component and the rows are positions, so a lane's unit has four codes of each
// of its four positions, twice.  A product's eight columns of values lie in one group of 32 components: their scale is the same
// and is multiplied into the weights on the left.
#ifndef LINMT_PAGES4_H_
#define LINMT_PAGES4_H_
#include <cstdint>

#ifdef __CUDACC__
#define LINMT_HD __host__ __device__ __forceinline__
#else
#define LINMT_HD inline
#endif

namespace linmt {
namespace pages4 {

constexpr int kTile = 16;                                     // positions of a tile
LINMT_HD constexpr int tile_bytes(int dim) { return 18 * dim; }
LINMT_HD constexpr int key_scales(int dim) { return 8 * dim; }
LINMT_HD constexpr int value_codes(int dim) { return 9 * dim; }
LINMT_HD constexpr int value_scales(int dim) { return 17 * dim; }

// Byte of the word that holds the eight key codes of components 8 w .. 8 w + 7 of position t.
LINMT_HD int key_word(int t, int w, int dim) { return t * (dim / 2) + 4 * ((w & 3) * (dim / 32) + (w >> 2)); }
// Byte of the 16-bit four of value codes of components 4 f .. 4 f + 3 of position t.
LINMT_HD int value_four(int t, int f, int dim) {
  const int i = f >> 4, h = (f >> 3) & 1, g = f & 7, a = t >> 3, c = (t & 7) >> 1, b = t & 1;
  return value_codes(dim) + 16 * ((i * 8 + g) * 4 + c) + 8 * a + 4 * h + 2 * b;
}
// Byte of the scale of components 32 s .. 32 s + 31 of position t, from the start of the keys' or the values' scales.
LINMT_HD int scale_at(int t, int s, int dim) { return 2 * (t * (dim / 32) + s); }

// Tile of a slot's position in the pool (head 0), -1 for a slot outside it.
LINMT_HD int64_t slot_page(int64_t slot, int n_pages, int page) {
  return slot < 0 || slot >= (int64_t)n_pages * page ? -1 : slot / page;
}
// Byte offset of tile `tile` (16 positions each) of a sentence whose table row is `table`; -1 where the table has no page of the pool.
LINMT_HD int64_t tile_offset(const int32_t* table, int tile, int tiles_per_page, int n_pages, int64_t stride_page, int dim) {
  const int32_t p = table[tile / tiles_per_page];
  return p < 0 || p >= n_pages ? -1 : (int64_t)p * stride_page + (int64_t)(tile % tiles_per_page) * tile_bytes(dim);
}

}  // namespace pages4
}  // namespace linmt
#endif
