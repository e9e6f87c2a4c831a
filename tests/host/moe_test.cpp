// Host-code test of the sparse MLP half (gdn_moe.cpp) under AddressSanitizer /
// UBSan, against the runtime stand-ins in fake_hip.cpp and fake_moe.cpp: the
// experts' packed layout, calls in several passes, what the entries refuse, and
// the executor's halves through prefills, steps, replacement and every error path.
// Exits 0 and prints "ALL OK" when every check holds.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include <hip/hip_runtime_api.h>

#include "gdn.h"
#include "gdn_common.h"

namespace gdn_fake {
extern bool capture;         // fake_hip.cpp: stream capture makes (empty) graphs
extern size_t malloc_bytes;  // fake_hip.cpp: size of the last device allocation
extern size_t malloc_limit;  // fake_hip.cpp: larger device allocations fail
extern int graphs_live, graphs_destroyed, graphs_made;
extern int moe_calls, route_calls, norm_calls, moe_rows, route_rows, norm_rows;  // fake_moe.cpp
}

static int g_checks = 0;
#define CHECK(cond)                                                                \
  do {                                                                             \
    ++g_checks;                                                                    \
    if (!(cond)) {                                                                 \
      std::fprintf(stderr, "FAILED %s:%d: %s (last error: %s)\n", __FILE__, __LINE__, \
                   #cond, gdn_last_error());                                       \
      return 1;                                                                    \
    }                                                                              \
  } while (0)

// n elements that end where their allocation does, aligned to `align`.
template <typename T>
static T* dev_alloc(std::vector<void*>& keep, size_t n, size_t align = 16) {
  void* p = nullptr;
  if (posix_memalign(&p, align, n * sizeof(T) ? n * sizeof(T) : 1) != 0) return nullptr;
  std::memset(p, 0, n * sizeof(T));
  keep.push_back(p);
  return static_cast<T*>(p);
}

struct Keep {
  std::vector<void*> all;
  ~Keep() {
    for (void* p : all) std::free(p);
  }
};

static gdn_moe_part make_part(Keep& k, int experts, int hidden, int inner) {
  gdn_moe_part p{};
  const size_t w = (size_t)experts * hidden * inner / 8, s = (size_t)experts * hidden * inner / 64;
  p.experts = experts;
  p.gate_w = dev_alloc<uint32_t>(k.all, w);
  p.gate_scales = dev_alloc<uint16_t>(k.all, s);
  p.gate_biases = dev_alloc<uint16_t>(k.all, s);
  p.up_w = dev_alloc<uint32_t>(k.all, w);
  p.up_scales = dev_alloc<uint16_t>(k.all, s);
  p.up_biases = dev_alloc<uint16_t>(k.all, s);
  p.down_w = dev_alloc<uint32_t>(k.all, w);
  p.down_scales = dev_alloc<uint16_t>(k.all, s);
  p.down_biases = dev_alloc<uint16_t>(k.all, s);
  return p;
}

static gdn_moe* make_moe(Keep& k, int hidden, int inner, std::vector<int> experts) {
  std::vector<gdn_moe_part> parts;
  for (int e : experts) parts.push_back(make_part(k, e, hidden, inner));
  gdn_moe* m = nullptr;
  if (gdn_moe_create(hidden, inner, (int)parts.size(), parts.data(), 64, 4, 0, nullptr, &m) != GDN_OK)
    return nullptr;
  return m;
}

static gdn_qlinear* make_qlinear(Keep& k, int K, std::vector<int32_t> rows) {
  std::vector<const uint32_t*> w;
  std::vector<const uint16_t*> s, b;
  for (int32_t n : rows) {
    w.push_back(dev_alloc<uint32_t>(k.all, (size_t)n * K / 8));
    s.push_back(dev_alloc<uint16_t>(k.all, (size_t)n * K / 64));
    b.push_back(dev_alloc<uint16_t>(k.all, (size_t)n * K / 64));
  }
  gdn_qlinear* q = nullptr;
  if (gdn_qlinear_create(K, (int)rows.size(), rows.data(), w.data(), s.data(), b.data(), 64, 4, 0,
                         nullptr, &q) != GDN_OK)
    return nullptr;
  return q;
}

// The packed arrays of odd shapes and several parts fit the layer's allocation, and
// calls of every size read and write what they were given, in one pass or more.
static int test_experts() {
  struct {
    int hidden, inner;
    std::vector<int> parts;
  } layers[] = {{128, 128, {1}}, {256, 128, {3, 1}}, {128, 384, {2, 1, 5}}, {640, 256, {4}}};
  for (const auto& l : layers) {
    Keep k;
    gdn_moe* m = make_moe(k, l.hidden, l.inner, l.parts);
    CHECK(m);
    int32_t hidden = 0, inner = 0, experts = 0, want = 0;
    for (int e : l.parts) want += e;
    CHECK(gdn_moe_dims(m, &hidden, &inner, &experts) == GDN_OK);
    CHECK(hidden == l.hidden && inner == l.inner && experts == want);
    for (int T : {1, 3, 64, 1500})
      for (int cols : {1, 3, 8}) {
        const int64_t xs = l.hidden + 8, os = l.hidden + 4;
        uint16_t* x = dev_alloc<uint16_t>(k.all, (size_t)(T - 1) * xs + l.hidden);
        uint16_t* out = dev_alloc<uint16_t>(k.all, (size_t)(T - 1) * os + l.hidden);
        int32_t* ids = dev_alloc<int32_t>(k.all, (size_t)T * cols);
        float* w = dev_alloc<float>(k.all, (size_t)T * cols);
        size_t bytes = 0;
        CHECK(gdn_moe_workspace_bytes(m, T, cols, &bytes) == GDN_OK);
        char* ws = dev_alloc<char>(k.all, bytes, 256);
        gdn_fake::moe_calls = gdn_fake::moe_rows = 0;
        CHECK(gdn_moe_forward(m, x, xs, T, cols, ids, w, out, os, ws, bytes, nullptr) == GDN_OK);
        const int pass = gdn::moe_pass_tokens(cols, xs);
        CHECK(gdn_fake::moe_rows == T && gdn_fake::moe_calls == (T + pass - 1) / pass);
        CHECK(gdn_moe_forward(m, x, xs, T, cols, ids, w, out, os, ws, bytes - 1, nullptr) ==
              GDN_ERR_INVALID);
      }
    CHECK(gdn_moe_destroy(m) == GDN_OK);
  }
  // no memory for the layer: nothing is left behind
  Keep k;
  gdn_moe_part p = make_part(k, 2, 128, 128);
  gdn_moe* m = nullptr;
  gdn_fake::malloc_limit = 100;
  CHECK(gdn_moe_create(128, 128, 1, &p, 64, 4, 0, nullptr, &m) == GDN_ERR_OOM && !m);
  gdn_fake::malloc_limit = ~(size_t)0;
  return 0;
}

static int test_route_and_norm() {
  Keep k;
  gdn_moe_route_desc d{60, 4, GDN_MOE_SIGMOID, 4, 2, 2, 1, 2.5f, 2, 1, 0};
  const int T = 37, cols = 61, stride = 70;
  uint16_t* logits = dev_alloc<uint16_t>(k.all, (size_t)(T - 1) * stride + cols);
  float* bias = dev_alloc<float>(k.all, 60);
  int32_t* ids = dev_alloc<int32_t>(k.all, T * 6);
  float* w = dev_alloc<float>(k.all, T * 6);
  CHECK(gdn_moe_route(&d, logits, stride, T, bias, ids, w, nullptr) == GDN_OK);
  CHECK(ids[T * 6 - 1] == 61);
  gdn_block_norm_desc n{};
  n.hidden = 264;
  n.scale = 1.0f;
  for (int f32 : {0, 1})
    for (int gate : {GDN_GATE_NONE, GDN_GATE_ROW, GDN_GATE_ELEMENT}) {
      n.h_f32 = f32;
      n.gate = gate;
      const int rows = 9;
      const int64_t s = 272;
      char* h = dev_alloc<char>(k.all, ((rows - 1) * s + 264) * (f32 ? 4 : 2));
      uint16_t* x = dev_alloc<uint16_t>(k.all, (rows - 1) * s + 264);
      uint16_t* g = dev_alloc<uint16_t>(k.all, gate == GDN_GATE_ROW ? rows : (rows - 1) * s + 264);
      uint16_t* wt = dev_alloc<uint16_t>(k.all, 264);
      CHECK(gdn_block_norm(&n, rows, h, s, x, s, wt, gate ? g : nullptr, gate == GDN_GATE_ROW ? 1 : s,
                           wt, h, s, x, s, nullptr) == GDN_OK);
    }
  return 0;
}

struct Stack {
  Keep k;
  gdn_pool* pool = nullptr;
  gdn_layer* layers[2] = {};
  gdn_kv* kv = nullptr;
  std::vector<gdn_qlinear*> qls;
  gdn_exec* ex = nullptr;
  static constexpr int hidden = 512, vocab = 1024, Hk = 16, Hv = 32, rows = 200;

  gdn_qlinear* ql(int K, std::vector<int32_t> n) {
    qls.push_back(make_qlinear(k, K, std::move(n)));
    return qls.back();
  }
  uint16_t* weights(size_t n) { return dev_alloc<uint16_t>(k.all, n); }

  // GatedDeltaNet, attention, GatedDeltaNet
  bool make() {
    const int D = 2 * Hk * 128 + Hv * 128, Hq = 16, Hkv = 2;
    gdn_pool_desc pd{2, 4, Hk, Hv, 128, 128, 4, 0};
    if (gdn_pool_create(&pd, &pool) != GDN_OK) return false;
    for (int l = 0; l < 2; ++l) {
      gdn_layer_desc ld{pool, l, ql(hidden, {D, Hv * 128, Hv, Hv}), ql(Hv * 128, {hidden}),
                        dev_alloc<float>(k.all, Hv), dev_alloc<float>(k.all, Hv),
                        weights((size_t)D * 4), weights(128), 1e-6f};
      if (gdn_layer_create(&ld, &layers[l]) != GDN_OK) return false;
    }
    gdn_kv_desc kd{1, 4, 24, 8, Hq, Hkv, 256, rows, 0, 0};
    if (gdn_kv_create(&kd, &kv) != GDN_OK) return false;
    gdn_exec_attn_layer al{1, ql(hidden, {Hq * 512 + 2 * Hkv * 256}), ql(Hq * 256, {hidden}),
                           weights(256), weights(256)};
    const uint16_t* norms[3] = {weights(hidden), weights(hidden), weights(hidden)};
    gdn_exec_desc ed{};
    ed.pool = pool;
    ed.num_layers = 2;
    ed.layers = layers;
    ed.input_norm_w = norms;
    ed.final_norm_w = weights(hidden);
    ed.rms_eps = 1e-6f;
    ed.embed = weights((size_t)vocab * hidden);
    ed.head = ql(hidden, {vocab});
    ed.max_batch = 4;
    ed.max_prompt = rows;
    ed.num_attn_layers = 1;
    ed.attn_layers = &al;
    ed.kv = kv;
    ed.rope_theta = 1e7f;
    ed.rotary_dim = 64;
    return gdn_exec_create(&ed, nullptr, &ex) == GDN_OK;
  }
  bool destroy() {
    bool ok = gdn_exec_destroy(ex) == GDN_OK;
    for (gdn_layer* l : layers) ok = gdn_layer_destroy(l) == GDN_OK && ok;
    for (gdn_qlinear* q : qls) ok = gdn_qlinear_destroy(q) == GDN_OK && ok;
    return gdn_kv_destroy(kv) == GDN_OK && gdn_pool_destroy(pool) == GDN_OK && ok;
  }
};

// Prefills and steps, captured and not, run the halves over their rows with the
// buffers of the executor's largest step; halves are replaced and taken away.
static int test_exec_halves(bool graphs) {
  gdn_fake::capture = graphs;
  gdn_fake::graphs_live = gdn_fake::graphs_destroyed = gdn_fake::graphs_made = 0;
  Stack s;
  CHECK(s.make());
  gdn_moe* a = make_moe(s.k, s.hidden, 128, {24, 1});
  gdn_moe* b = make_moe(s.k, s.hidden, 384, {8});
  CHECK(a && b);
  gdn_qlinear* gate = s.ql(s.hidden, {32});
  gdn_moe_route_desc ra{24, 4, GDN_MOE_SOFTMAX, 1, 1, 1, 1, 1.0f, 1, 1, 0};
  gdn_moe_route_desc rb{8, 3, GDN_MOE_SIGMOID, 1, 1, 1, 1, 1.0f, 0, 0, 0};
  float* bias = dev_alloc<float>(s.k.all, 8);
  const gdn_exec_moe halves[3] = {{0, s.weights(s.hidden), gate, &ra, nullptr, a},
                                  {2, s.weights(s.hidden), gate, &rb, bias, b},
                                  {1, s.weights(s.hidden), gate, &ra, nullptr, a}};
  std::vector<int32_t> p(s.rows, 7);
  const uint64_t ids[2] = {1, 2};
  uint32_t toks[2] = {1, 2}, next[2], t = 0;
  for (int n : {3, 0, 2, 1}) {
    CHECK(gdn_exec_set_moe(s.ex, n, n ? halves : nullptr) == GDN_OK);
    CHECK(gdn_fake::graphs_live == 0);
    gdn_fake::moe_rows = 0;
    CHECK(gdn_exec_prefill(s.ex, 1, p.data(), s.rows, &t) == GDN_OK);
    CHECK(gdn_fake::moe_rows == n * s.rows);
    CHECK(gdn_exec_prefill(s.ex, 2, p.data(), 5, &t) == GDN_OK);
    gdn_fake::moe_rows = 0;
    CHECK(gdn_exec_decode_batch(s.ex, ids, toks, 2, next) == GDN_OK);
    CHECK(gdn_fake::moe_rows == n * 2);
    const int made = gdn_fake::graphs_made;
    CHECK(gdn_exec_decode_batch(s.ex, ids, toks, 2, next) == GDN_OK);
    CHECK(gdn_fake::graphs_made == made && (made > 0) == graphs);
    gdn_fake::malloc_bytes = 0;
    CHECK(gdn_exec_set_moe(s.ex, n, n ? halves : nullptr) == GDN_ERR_INVALID);
    CHECK(std::strstr(gdn_last_error(), "holds 2 sequences"));
    CHECK(gdn_fake::malloc_bytes == 0);  // refused before anything is allocated
    for (uint64_t id : ids) CHECK(gdn_exec_release(s.ex, id) == GDN_OK);
  }
  // what every later step would fail at is refused here; the halves stay as they were
  gdn_exec_moe odd = halves[1];
  odd.bias = reinterpret_cast<const float*>(reinterpret_cast<const char*>(bias) + 2);
  CHECK(gdn_exec_set_moe(s.ex, 1, &odd) == GDN_ERR_INVALID);
  // no memory for the buffers: the same
  gdn_fake::malloc_limit = 1000;
  CHECK(gdn_exec_set_moe(s.ex, 3, halves) == GDN_ERR_OOM);
  gdn_fake::malloc_limit = ~(size_t)0;
  gdn_fake::moe_rows = 0;
  CHECK(gdn_exec_prefill(s.ex, 1, p.data(), 9, &t) == GDN_OK);
  CHECK(gdn_fake::moe_rows == 9);
  CHECK(s.destroy());
  CHECK(gdn_moe_destroy(a) == GDN_OK && gdn_moe_destroy(b) == GDN_OK);
  CHECK(gdn_fake::graphs_live == 0);
  gdn_fake::capture = false;
  return 0;
}

int main() {
  if (test_experts() || test_route_and_norm() || test_exec_halves(false) || test_exec_halves(true))
    return 1;
  std::printf("ALL OK (%d checks)\n", g_checks);
  return 0;
}
