// How attention over the 8-bit cache cuts a row's pages (gdn_common.h), against the mask's
// definition: the pages of an item are the ones that hold a key that it sees, each once and
// in order, and its pieces take each of them once and have room for their results.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "gdn_common.h"

namespace {

long checks = 0;

[[noreturn]] void fail(const char* what, int per, int pos, int fresh, int window, int pf, int pieces,
                       int item) {
  std::printf("FAILED: %s: %d tokens an item, %d cached, %d new, window %d, prefix %d, %d pieces, "
              "item %d\n", what, per, pos, fresh, window, pf, pieces, item);
  std::exit(1);
}

void row(int per, int pos, int fresh, int window, int pf, int pieces, int unit, int least) {
  const int total = pos + fresh;
  const gdn::Kv8Cut c = gdn::kv8_cut(pos, fresh, window, pf, per, pieces, unit, least);
  if (c.items != (fresh + per - 1) / per || c.n < 1 || c.n > pieces || c.cp % unit != 0)
    fail("the cut", per, pos, fresh, window, pf, pieces, -1);
  for (int g = 0; g < c.items; ++g) {
    const int p0 = pos + g * per, p1 = std::min(p0 + per, total) - 1;
    const gdn::Kv8Span s = gdn::kv8_span(p0, p1, window, pf, total);
    // pages that hold a key seen from p0 .. p1: below the prefix, or above the first one's
    // window and up to the last one
    std::vector<int> want;
    for (int page = 0; page * 64 < total; ++page) {
      const int a = page * 64, b = std::min(a + 63, total - 1);
      const bool seen = a < pf || (a <= p1 && (window == 0 || b > p0 - window));
      if (seen) want.push_back(page);
    }
    if (s.count() != (int)want.size()) fail("the count", per, pos, fresh, window, pf, pieces, g);
    for (int v = 0; v < s.count(); ++v)
      if (s.page(v) != want[v]) fail("a page", per, pos, fresh, window, pf, pieces, g);
    int at = 0;  // pieces are [i * cp, end), or empty
    for (int i = 0; i < c.n; ++i) {
      const int end = gdn::kv8_piece_end(c, i, s.count());
      if (i * c.cp >= end) continue;
      if (i * c.cp != at) fail("pieces", per, pos, fresh, window, pf, pieces, g);
      at = end;
    }
    if (at != s.count()) fail("pages that no piece reads", per, pos, fresh, window, pf, pieces, g);
    ++checks;
  }
}

}  // namespace

int main() {
  row(128, 1000, 1537, 1900, 0, 4, 1, 8);
  row(128, 1, 1025, 896, 0, 5, 1, 8);
  std::mt19937 rng(1);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  for (int G = 1; G <= 16; ++G) {
    const int tile = gdn::kKv8TileWaves * (32 / G), group = 16 / G;
    for (int i = 0; i < 6000; ++i) {
      const int pos = upto(i % 3 ? 1500 : 100), window = i % 4 ? 1 + upto(2000) : 0;
      const int pf = i % 5 ? 0 : upto(900);
      const int fresh = 1 + upto(1700), few = 1 + upto(gdn::kKv8TileTokens - 2);
      row(tile, pos, fresh, window, std::min(pf, pos + fresh), 2 + upto(20), 1, 8);
      row(tile, pos, few, window, std::min(pf, pos + few), 2 + upto(200), 1, 8);
      const int n = 1 + upto(i % 7 ? 40 : 4095), Hkv = 1 + upto(i % 6 ? 8 : 255), groups = (few + group - 1) / group;
      row(group, pos, few, window, std::min(pf, pos + few), gdn::kv8_chunks(n, Hkv, groups),
          gdn::kv8_chunk_waves(n, Hkv), 1);
      // room for the partial results of every row
      const int chunks = gdn::kv8_chunks(n, Hkv, groups), room = gdn::kv8_row_parts(n, Hkv);
      if ((chunks > 1 && groups * chunks > room) || n * Hkv * room > gdn::kKv8Waves)
        fail("room", group, pos, few, window, n, chunks, room);
    }
  }
  std::printf("%ld items\nALL OK\n", checks);
  return 0;
}
