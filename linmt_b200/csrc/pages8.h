// pages8.h -- where a pool of 8-bit pages keeps what (the form is in include/linmt_decoder.h).  Host and device: the tests
// check the same functions on the CPU.
//
// A block's codes lie as tcgen05.mma wants its left operand in shared memory without a swizzle: eight rows of 16 bytes one behind the other.  Keys: a row is
// a position and the 16 bytes are components.  Values: a row is a component and the 16 bytes are the block's positions.  So the attention
// kernel copies blocks as they are and multiplies, and nothing is unpacked.
#ifndef LINMT_PAGES8_H_
#define LINMT_PAGES8_H_
#include <cstdint>

#ifdef __CUDACC__
#define LINMT_HD8 __host__ __device__ __forceinline__
#else
#define LINMT_HD8 inline
#endif

namespace linmt {
namespace pages8 {

constexpr int kBlock = 16;                                    // positions of a block
LINMT_HD8 constexpr int block_bytes(int dim) { return 32 * dim + 16; }
LINMT_HD8 constexpr int value_codes(int dim) { return 16 * dim; }
LINMT_HD8 constexpr int scales(int dim) { return 32 * dim; }  // two floats: keys, values

// Byte of the 16 key codes of components 16 u .. 16 u + 15 of position t.
LINMT_HD8 constexpr int key_unit(int t, int u, int dim) { return (t >> 3) * 8 * dim + u * 128 + (t & 7) * 16; }
// Byte of the 16 value codes (one of each position) of component c.
LINMT_HD8 constexpr int value_unit(int c, int dim) { return value_codes(dim) + 16 * c; }

// Page of a slot, -1 for a slot outside the pool.
LINMT_HD8 int64_t slot_page(int64_t slot, int n_pages, int page) {
  return slot < 0 || slot >= (int64_t)n_pages * page ? -1 : slot / page;
}
// Byte offset of a slot's block in the pool (head 0), -1 for a slot outside it.
LINMT_HD8 int64_t slot_block(int64_t slot, int n_pages, int page, int64_t stride_page, int dim) {
  const int64_t p = slot_page(slot, n_pages, page);
  return p < 0 ? -1 : p * stride_page + (slot - p * page) / kBlock * block_bytes(dim);
}
// Byte offset of block `block` (16 positions each) of a sentence whose table row is `table`; -1 where the table has no page of the pool.
LINMT_HD8 int64_t block_offset(const int32_t* table, int block, int blocks_per_page, int n_pages, int64_t stride_page, int dim) {
  const int32_t p = table[block / blocks_per_page];
  return p < 0 || p >= n_pages ? -1 : (int64_t)p * stride_page + (int64_t)(block % blocks_per_page) * block_bytes(dim);
}

// The runs of a write: of 32 neighbours in a list of slots, bit l of `goes_on` says that slot l is in the block of slot l - 1 and follows it.
LINMT_HD8 bool follows(int64_t before, int64_t slot) { return before >= 0 && slot == before + 1 && (slot & (kBlock - 1)) != 0; }

}  // namespace pages8
}  // namespace linmt
#endif
