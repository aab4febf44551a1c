// The form of a 4-bit page's tile and the look-up of tiles, on the CPU.  Prints one line for each check that fails.
#include <cstdio>
#include <vector>

#include "pages4.h"

int main() {
  using namespace linmt::pages4;
  int bad = 0;
  auto fail = [&](const char* what, int a, int b) { std::printf("%s: %d %d\n", what, a, b); ++bad; };
  for (int dim : {64, 128}) {
    std::vector<int> owner(tile_bytes(dim), -1);
    auto take = [&](int at, int bytes, int who) {
      for (int i = 0; i < bytes; ++i) {
        if (at + i < 0 || at + i >= tile_bytes(dim)) { fail("outside the tile", at + i, who); return; }
        if (owner[at + i] != -1) fail("taken twice", at + i, who);
        owner[at + i] = who;
      }
    };
    for (int t = 0; t < kTile; ++t) {
      for (int w = 0; w < dim / 8; ++w) take(key_word(t, w, dim), 4, 1);
      for (int f = 0; f < dim / 4; ++f) take(value_four(t, f, dim), 2, 2);
      for (int s = 0; s < dim / 32; ++s) {
        take(key_scales(dim) + scale_at(t, s, dim), 2, 3);
        take(value_scales(dim) + scale_at(t, s, dim), 2, 4);
      }
    }
    for (int i = 0; i < tile_bytes(dim); ++i)
      if (owner[i] == -1) fail("free", i, dim);
    // lanes 4 g + c of the attention kernel: keys of position 8 j + g, words c dim / 32 + group; values 16 bytes a lane
    for (int lane = 0; lane < 32; ++lane) {
      const int g = lane >> 2, c = lane & 3;
      for (int j = 0; j < 2; ++j)
        for (int gr = 0; gr < dim / 32; ++gr)
          if (key_word(8 * j + g, 4 * gr + c, dim) != (8 * j + g) * (dim / 2) + c * (dim / 8) + 4 * gr) fail("key", lane, gr);
      for (int gr = 0; gr < dim / 32; ++gr)
        for (int k = 0; k < 4; ++k) {
          const int t = 2 * c + (k & 1) + 8 * (k >> 1);
          if (value_four(t, 8 * gr + g, dim) != value_codes(dim) + 16 * ((gr >> 1) * 32 + lane) + 8 * (k >> 1) + 4 * (gr & 1) + 2 * (k & 1)) fail("value", lane, gr);
        }
    }
    // look-ups: pages that are none of the pool's, offsets past 32 bits
    const int32_t table[4] = {2, -1, 7, 2000000};
    const int64_t stride = 8ll * 4 * tile_bytes(dim);
    if (tile_offset(table, 3, 4, 3, stride, dim) != 2 * stride + 3 * tile_bytes(dim)) fail("page 2", dim, 0);
    if (tile_offset(table, 4, 4, 3, stride, dim) != -1 || tile_offset(table, 7, 4, 3, stride, dim) != -1) fail("page -1", dim, 0);
    if (tile_offset(table, 8, 4, 7, stride, dim) != -1 || tile_offset(table, 8, 4, 8, stride, dim) != 7 * stride) fail("page 7", dim, 0);
    if (tile_offset(table, 13, 4, 2000001, stride, dim) != 2000000 * stride + tile_bytes(dim)) fail("far page", dim, 0);
  }
  if (slot_page(-1, 5, 32) != -1 || slot_page(160, 5, 32) != -1 || slot_page(159, 5, 32) != 4 || slot_page(0, 5, 32) != 0) fail("slot", 0, 0);
  if (slot_page(1ll << 40, 5, 32) != -1 || slot_page((1ll << 31) * 48 + 50, 2147483647, 128) != ((1ll << 31) * 48 + 50) / 128) fail("far slot", 0, 0);
  return bad != 0;
}
