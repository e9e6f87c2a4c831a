// Stand-ins for the sparse MLP half's launches (gdn_moe.hip, gdn_route.hip,
// gdn_norm.hip), beside fake_hip.cpp. They compute nothing, but read every
// element that the kernels read and write every one that they write, so that
// AddressSanitizer sees a buffer that gdn_moe.cpp made too small or a pointer
// that it placed wrongly, also when a captured launch is replayed. Workspace sizes
// stand for the library's.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstring>
#include <functional>
#include <vector>

#include "gdn_common.h"

namespace gdn_fake {
extern std::vector<std::function<void()>>* recording;  // fake_hip.cpp: the capture in progress
int moe_calls = 0, route_calls = 0, norm_calls = 0;
int moe_rows = 0, route_rows = 0, norm_rows = 0;  // of all calls
}

namespace gdn {
namespace {

// Reads n bytes.
unsigned touch(const void* p, size_t n) {
  unsigned s = 0;
  for (size_t i = 0; i < n; ++i) s += static_cast<const unsigned char*>(p)[i];
  return s;
}
volatile unsigned sink;

void route(const MoeRouteArgs& a) {
  ++gdn_fake::route_calls;
  gdn_fake::route_rows += a.T;
  const int cols = a.d.num_experts + (a.d.shared_gate ? 1 : 0), k = a.d.top_k + a.d.num_shared;
  const size_t elem = a.d.logits_f32 ? 4 : 2;
  for (int t = 0; t < a.T; ++t) {
    sink = touch(static_cast<const char*>(a.logits) + t * a.stride * elem, cols * elem);
    for (int j = 0; j < k; ++j) {
      a.ids[(size_t)t * k + j] = j < a.d.top_k ? j : a.d.num_experts + j - a.d.top_k;
      a.weights[(size_t)t * k + j] = 1.0f / k;
    }
  }
  if (a.bias) sink = touch(a.bias, a.d.num_experts * 4);
}

void experts(const MoeArgs& a) {
  ++gdn_fake::moe_calls;
  gdn_fake::moe_rows += a.T;
  const size_t terms = (size_t)a.hidden * a.inner * a.experts;
  sink = touch(a.w1, terms) + touch(a.w2, terms / 2) + touch(a.sb1, terms / 8) +
         touch(a.sb2, terms / 16) + touch(a.bound, 12 * (size_t)a.experts);
  std::memset(a.workspace, 3, moe_workspace_bytes(a.hidden, a.inner, a.experts, a.T, a.k));
  for (int t = 0; t < a.T; ++t) {
    sink = touch(a.x + t * a.xs, 2 * (size_t)a.hidden) + touch(a.ids + (size_t)t * a.k, 4 * (size_t)a.k) +
           touch(a.weights + (size_t)t * a.k, 4 * (size_t)a.k);
    std::memset(a.out + t * a.os, 0, 2 * (size_t)a.hidden);
  }
}

template <typename F>
void run(F f) {
  if (gdn_fake::recording)
    gdn_fake::recording->push_back(f);
  else
    f();
}

}  // namespace

hipError_t launch_moe_route(const MoeRouteArgs& a) {
  run([=] { route(a); });
  return hipSuccess;
}

hipError_t launch_moe_pack(const MoePackArgs& a) {
  const size_t words = (size_t)a.experts * a.n * (a.k / 8), groups = (size_t)a.experts * a.n * (a.k / 64);
  sink = touch(a.w, 4 * words) + touch(a.s, 2 * groups) + touch(a.b, 2 * groups);
  const int P = a.k / 128;
  for (int e = 0; e < a.experts; ++e)
    for (int f = 0; f < a.n / 16; ++f) {
      const size_t at = ((size_t)e * a.frags + a.fmul * f + a.fofs) * P;
      std::memset(static_cast<char*>(a.wp) + at * 1024, 1, (size_t)P * 1024);
      std::memset(a.sb + at * 32, 1, (size_t)P * 128);
    }
  return hipSuccess;
}

hipError_t launch_moe_bound(const MoePackArgs& a, bool, float* bound) {
  for (int e = 0; e < a.experts; ++e) {
    if (bound[e] != 0.0f) return hipErrorInvalidValue;  // zeros before
    bound[e] = 1.0f;
  }
  return hipSuccess;
}

int moe_pass_tokens(int k, int64_t) { return 4096 / k; }
size_t moe_workspace_bytes(int hidden, int inner, int experts, int T, int k) {
  const size_t entries = std::min<size_t>((size_t)T * k, 4096);
  return entries * (hidden * 4 + inner * 2) + (size_t)experts * 16 + 256;
}

hipError_t launch_moe(const MoeArgs& a) {
  for (int i = 0; i < 3 * a.experts; ++i)
    if (a.bound[i] != 1.0f) return hipErrorInvalidValue;  // every matrix has its bound
  run([=] { experts(a); });
  return hipSuccess;
}

hipError_t launch_block_norm(const BlockNormArgs& a) {
  ++gdn_fake::norm_calls;
  gdn_fake::norm_rows += a.n;
  const size_t hid = a.d.hidden, hb = a.d.h_f32 ? 4 : 2;
  for (int i = 0; i < a.n; ++i) {
    sink = touch(static_cast<const char*>(a.h) + i * a.h_stride * hb, hid * hb) +
           touch(a.x + i * a.x_stride, 2 * hid);
    if (a.gate) sink = touch(a.gate + i * a.gate_stride, a.d.gate == GDN_GATE_ROW ? 2 : 2 * hid);
    std::memset(static_cast<char*>(a.h_out) + i * a.h_out_stride * hb, 0, hid * hb);
    if (a.hn) std::memset(a.hn + i * a.hn_stride, 0, 2 * hid);
  }
  if (a.post_w) sink = touch(a.post_w, 2 * hid);
  if (a.pre_w) sink = touch(a.pre_w, 2 * hid);
  return hipSuccess;
}

}  // namespace gdn
