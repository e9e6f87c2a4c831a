// Host code of the 8-bit cache and the rotary positions under AddressSanitizer / UBSan.
//
// How attention cuts a row's pages (gdn_common.h), against the mask's definition: the pages of
// an item are the ones that hold a key that it sees, each once and in order, and its pieces take
// each of them once and have room for their results.
//
// The entries (gdn_kv8.cpp), against the runtime stand-ins in fake_hip.cpp and fake_kv8.cpp: the
// device arrays' places and sizes, what is refused, allocations that fail.
// Exits 0 and prints "ALL OK" when every check holds.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "gdn.h"
#include "gdn_common.h"

namespace gdn_fake {
extern size_t malloc_bytes;  // fake_hip.cpp: size of the last device allocation
extern size_t malloc_limit;  // fake_hip.cpp: larger device allocations fail
extern int step_calls, append_calls, gather_calls, attn_calls, rope_calls;  // fake_kv8.cpp
extern gdn::Kv8Plan plan;
extern gdn::Kv8AttnArgs attn8;
}

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

#define CHECK(cond)                                                                  \
  do {                                                                               \
    ++checks;                                                                        \
    if (!(cond)) {                                                                   \
      std::printf("FAILED %s:%d: %s (last error: %s)\n", __FILE__, __LINE__, #cond, \
                  gdn_last_error());                                                 \
      std::exit(1);                                                                  \
    }                                                                                \
  } while (0)

// n elements that end where their allocation does
template <typename T>
struct Dev {
  T* at = nullptr;
  explicit Dev(size_t n) {
    if (posix_memalign(reinterpret_cast<void**>(&at), 16, n * sizeof(T) ? n * sizeof(T) : 1)) std::abort();
    std::memset(at, 0, n * sizeof(T));
  }
  Dev(const Dev&) = delete;
  ~Dev() { std::free(at); }
  operator T*() const { return at; }
};

void cache(int layers, int slots, int pages, int per_slot, int Hq, int Hkv, int D, int tokens) {
  const gdn_kv8_desc d{layers, slots, pages, per_slot, Hq, Hkv, D, tokens, 0};
  gdn_kv8* kv = nullptr;
  CHECK(gdn_kv8_create(&d, &kv) == GDN_OK && kv);
  gdn_kv8_desc back{};
  CHECK(gdn_kv8_describe(kv, &back) == GDN_OK && std::memcmp(&back, &d, sizeof(d)) == 0);
  gdn_kv8_view view{};
  CHECK(gdn_kv8_views(kv, &view) == GDN_OK && *view.free_count == pages);
  for (int i = 0; i < pages; ++i) CHECK(view.free_pages[i] == pages - 1 - i);
  for (int i = 0; i < slots * per_slot; ++i) CHECK(view.table[i] == -1);
  uint32_t flags = 1;
  CHECK(gdn_kv8_check(kv, nullptr, &flags) == GDN_OK && flags == 0);
  const size_t row = (size_t)Hkv * D, qrow = (size_t)Hq * D;
  const gdn_kv8_attn_desc a{};
  Dev<uint16_t> none(8);
  CHECK(gdn_kv8_append(kv, 0, none, row, none, row, nullptr) == GDN_ERR_INVALID);  // no step
  for (const int n : {1, 4096})
    for (const int T : {0, 1, tokens}) {
      Dev<int32_t> s(n), l(n), t(n), out(n), prefix(n);
      const int calls = gdn_fake::step_calls;
      CHECK(gdn_kv8_step(kv, n, s, l, t, n == 1 ? nullptr : (int32_t*)out, T, 0, nullptr) == GDN_OK);
      CHECK(gdn_fake::step_calls == calls + 1 && gdn_fake::plan.n == n && gdn_fake::plan.T == T &&
            gdn_fake::plan.max_row == T);
      Dev<uint16_t> k(T * row), v(T * row), q(T * qrow), g(T * qrow), o(T * qrow);
      Dev<float> slopes(Hq);
      for (int layer = 0; layer < layers; ++layer) {
        CHECK(gdn_kv8_append(kv, layer, k, row, v, row, nullptr) == GDN_OK);
        CHECK(gdn_kv8_attention(kv, layer, &a, q, qrow, D, slopes, prefix, g, qrow, D, o, qrow, D,
                                nullptr) == GDN_OK);
        CHECK(gdn_kv8_attention(kv, layer, &a, q, D, T * D, nullptr, nullptr, nullptr, 0, 0, o, D,
                                (int64_t)T * D, nullptr) == GDN_OK || T == 0);  // heads first
      }
      CHECK(gdn_kv8_append(kv, layers, k, row, v, row, nullptr) == GDN_ERR_INVALID || T == 0);
      if (T > 1) {
        // rows and planes that run into each other, numbers that are none
        if (Hkv > 1) CHECK(gdn_kv8_append(kv, 0, k, row - 8, v, row, nullptr) == GDN_ERR_INVALID);
        if (Hkv > 1) CHECK(gdn_kv8_append(kv, 0, k, row, v, D, nullptr) == GDN_ERR_INVALID);
        CHECK(gdn_kv8_append(kv, 0, k, row + 4, v, row, nullptr) == GDN_ERR_INVALID);
        CHECK(gdn_kv8_append(kv, 0, k + 4, row, v, row, nullptr) == GDN_ERR_INVALID);
        if (Hq > 1)
          CHECK(gdn_kv8_attention(kv, 0, &a, q, qrow, D, nullptr, nullptr, nullptr, 0, 0, o, D,
                                  (int64_t)(T - 1) * D, nullptr) == GDN_ERR_INVALID);
        for (const float cap : {-1.0f, 1e-31f, 1e31f, INFINITY, NAN}) {
          const gdn_kv8_attn_desc bad{0.0f, cap, 0};
          CHECK(gdn_kv8_attention(kv, 0, &bad, q, qrow, D, nullptr, nullptr, nullptr, 0, 0, o, qrow, D,
                                  nullptr) == GDN_ERR_INVALID);
        }
      }
      for (const int m : {0, 1, 70}) {
        Dev<int32_t> map(m);
        Dev<uint16_t> ko(m * row), vo(m * row);
        CHECK(gdn_kv8_gather(kv, 0, m, map, ko, row, vo, row, nullptr) == GDN_OK);
        CHECK(gdn_kv8_gather(kv, 0, m, map, nullptr, 0, vo, row, nullptr) == GDN_OK);
        if (m == 1) CHECK(gdn_kv8_gather(kv, 0, m, map, ko, 0, vo, 8, nullptr) == GDN_OK);
        if (m > 1 && Hkv > 1)
          CHECK(gdn_kv8_gather(kv, 0, m, map, ko, D, nullptr, 0, nullptr) == GDN_ERR_INVALID);
      }
    }
  CHECK(gdn_kv8_destroy(kv) == GDN_OK);
  // every allocation that may fail
  size_t most = 0, least = ~(size_t)0;
  for (const size_t bytes : {(size_t)2 * Hkv * 64 * D * pages, (size_t)8 * Hkv * pages}) {
    most = bytes > most ? bytes : most;
    least = bytes < least ? bytes : least;
  }
  for (const size_t limit : {(size_t)0, least - 1, least, most - 1, most}) {
    gdn_fake::malloc_limit = limit;
    const gdn_status st = gdn_kv8_create(&d, &kv);
    CHECK(st == GDN_OK || (st == GDN_ERR_OOM && kv == nullptr));
    if (st == GDN_OK) gdn_kv8_destroy(kv);
  }
  gdn_fake::malloc_limit = ~(size_t)0;
}

void rope(int D, int rot, int f32) {
  for (int scaling = GDN_ROPE_NONE; scaling <= GDN_ROPE_BANDS; ++scaling) {
    const gdn_rope_desc d{D, rot, scaling & 1, scaling, 1e4f, 4.0f, 4096.0f, 32.0f, 1.0f, 0.0f};
    gdn_rope* r = nullptr;
    CHECK(gdn_rope_create(&d, 0, &r) == GDN_OK && r);
    const int T = 3, Hq = 4, Hk = 1;
    Dev<int32_t> pos(T);
    Dev<float> q(T * Hq * D), k(T * Hk * D);
    Dev<uint16_t> w(D);
    const gdn_rope_rows qr{q, q, Hq, Hq * D, D, Hq * D, D, w}, kr{k, k, Hk, Hk * D, D, Hk * D, D, nullptr};
    CHECK(gdn_rope_forward(r, T, pos, &qr, &kr, f32, 1e-6f, 0, nullptr) == GDN_OK);
    CHECK(gdn_rope_forward(r, T, pos, &kr, nullptr, f32, 0.0f, 1, nullptr) == GDN_OK);
    gdn_rope_rows bad = qr;
    bad.out_head_stride = D - 8;
    CHECK(gdn_rope_forward(r, T, pos, &bad, nullptr, f32, 0.0f, 0, nullptr) == GDN_ERR_INVALID);
    bad = qr;
    bad.out_stride = bad.in_stride = D;  // tokens that run into each other
    CHECK(gdn_rope_forward(r, T, pos, &bad, nullptr, f32, 0.0f, 0, nullptr) == GDN_ERR_INVALID);
    CHECK(gdn_rope_destroy(r) == GDN_OK);
    gdn_fake::malloc_limit = 0;
    CHECK(gdn_rope_create(&d, 0, &r) == GDN_ERR_OOM && r == nullptr);
    gdn_fake::malloc_limit = ~(size_t)0;
  }
}

}  // namespace

int main() {
  cache(1, 1, 1, 1, 1, 1, 64, 1);
  cache(2, 3, 7, 5, 6, 2, 64, 33);
  cache(1, 9, 4, 11, 16, 1, 256, 20);
  cache(3, 2, 5, 3, 4, 4, 128, 70);
  for (const int D : {8, 64, 520 - 8}) {
    rope(D, D, 0);
    rope(D, D / 4 * 2, 1);
    rope(D, 0, 0);
  }
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
  std::printf("%ld checks\nALL OK\n", checks);
  return 0;
}
