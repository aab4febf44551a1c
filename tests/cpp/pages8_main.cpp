// The form of an 8-bit page's block, the look-up of blocks and the runs of a write, on the CPU.  Prints one line for each check that fails.
#include <cstdio>
#include <vector>

#include "pages8.h"

int main() {
  using namespace linmt::pages8;
  int bad = 0;
  auto fail = [&](const char* what, int a, int b) { std::printf("%s: %d %d\n", what, a, b); ++bad; };
  for (int dim : {64, 128}) {
    std::vector<int> owner(block_bytes(dim), -1);
    auto take = [&](int at, int bytes, int who) {
      for (int i = 0; i < bytes; ++i) {
        if (at + i < 0 || at + i >= block_bytes(dim)) { fail("outside the block", at + i, who); return; }
        if (owner[at + i] != -1) fail("taken twice", at + i, who);
        owner[at + i] = who;
      }
    };
    for (int t = 0; t < kBlock; ++t)
      for (int u = 0; u < dim / 16; ++u) take(key_unit(t, u, dim), 16, 1);
    for (int c = 0; c < dim; ++c) take(value_unit(c, dim), 16, 2);
    take(scales(dim), 16, 3);
    for (int i = 0; i < block_bytes(dim); ++i)
      if (owner[i] == -1) fail("free", i, dim);
    if (block_bytes(dim) % 16 || value_codes(dim) % 128) fail("alignment", dim, 0);
    // cores of eight rows of 16 bytes: of keys eight positions, of values eight components, one row behind the other
    for (int t = 0; t < kBlock; ++t)
      for (int u = 0; u < dim / 16; ++u)
        if (key_unit(t, u, dim) != t / 8 * 8 * dim + u * 128 + t % 8 * 16) fail("key", t, u);
    for (int c = 0; c < dim; ++c)
      if (value_unit(c, dim) - value_codes(dim) != c / 8 * 128 + c % 8 * 16) fail("value", c, dim);
    // look-ups: pages that are none of the pool's, offsets past 32 bits
    const int32_t table[4] = {2, -1, 7, 2000000};
    const int64_t stride = 8ll * 4 * block_bytes(dim);
    if (block_offset(table, 3, 4, 3, stride, dim) != 2 * stride + 3 * block_bytes(dim)) fail("page 2", dim, 0);
    if (block_offset(table, 4, 4, 3, stride, dim) != -1 || block_offset(table, 7, 4, 3, stride, dim) != -1) fail("page -1", dim, 0);
    if (block_offset(table, 8, 4, 7, stride, dim) != -1 || block_offset(table, 8, 4, 8, stride, dim) != 7 * stride) fail("page 7", dim, 0);
    if (block_offset(table, 13, 4, 2000001, stride, dim) != 2000000 * stride + block_bytes(dim)) fail("far page", dim, 0);
    if (slot_block(-1, 5, 32, stride, dim) != -1 || slot_block(160, 5, 32, stride, dim) != -1 || slot_block(159, 5, 32, stride, dim) != 4 * stride + block_bytes(dim)) fail("slot", dim, 0);
    if (slot_block((1ll << 31) * 48 + 50, 2147483647, 128, stride, dim) != ((1ll << 31) * 48 + 50) / 128 * stride + ((1ll << 31) * 48 + 50) % 128 / 16 * block_bytes(dim)) fail("far slot", dim, 0);
  }
  if (slot_page(-1, 5, 32) != -1 || slot_page(160, 5, 32) != -1 || slot_page(159, 5, 32) != 4 || slot_page(0, 5, 32) != 0 || slot_page(1ll << 40, 5, 32) != -1) fail("page", 0, 0);
  if (follows(-1, 0) || follows(15, 16) || follows(3, 5) || follows(5, 4) || follows(7, -1) || !follows(0, 1) || !follows(30, 31)) fail("runs", 0, 0);
  return bad != 0;
}
