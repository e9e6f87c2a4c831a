// Stand-ins for the launches of the 8-bit cache and the rotary positions (gdn_kv8.hip,
// gdn_attn8.hip, gdn_rope.hip), beside fake_hip.cpp. They compute nothing, but read every element
// that the kernels may read and write every one that they may write, so that AddressSanitizer
// sees an array that gdn_kv8.cpp made too small or placed on another one's end.
#include <hip/hip_runtime.h>

#include <cstring>

#include "gdn_common.h"

namespace gdn_fake {
int step_calls = 0, append_calls = 0, gather_calls = 0, attn_calls = 0, rope_calls = 0;
gdn::Kv8Plan plan;       // of the last step
gdn::Kv8AttnArgs attn8;  // of the last attention
}

namespace gdn {
namespace {

unsigned touch(const void* p, size_t n) {
  unsigned s = 0;
  for (size_t i = 0; i < n; ++i) s += static_cast<const unsigned char*>(p)[i];
  return s;
}
volatile unsigned sink;

// Rows of `heads` heads of `dim` elements of `elem` bytes; written with `value`, or read.
void rows(const void* p, int64_t tokens, int64_t stride, int64_t head_stride, int heads, int dim,
          int elem, int value = -1) {
  for (int64_t t = 0; t < tokens; ++t)
    for (int h = 0; h < heads; ++h) {
      char* const at = const_cast<char*>(static_cast<const char*>(p)) + (t * stride + h * head_stride) * elem;
      if (value < 0)
        sink += touch(at, (size_t)dim * elem);
      else
        std::memset(at, value, (size_t)dim * elem);
    }
}

void tables(const Kv8Plan& p) {
  sink += touch(p.table, sizeof(int32_t) * p.num_slots * p.max_pages) +
          touch(p.owned, sizeof(int32_t) * p.num_slots) + touch(p.rows, sizeof(Kv8Row) * p.n) +
          touch(p.blocks, sizeof(int32_t) * (p.n + 1)) + touch(p.tiles, sizeof(int32_t) * p.n) +
          touch(p.tok_row, sizeof(int32_t) * p.T);
}

void pages(const Kv8Plan& p, const uint8_t* bytes, const int32_t* exps) {
  const size_t heads = (size_t)p.num_pages * 2 * p.Hkv;
  sink += touch(bytes, heads * 64 * p.D) + touch(exps, heads * sizeof(int32_t));
}

}  // namespace

hipError_t launch_kv8_step(const Kv8StepArgs& a) {
  ++gdn_fake::step_calls;
  gdn_fake::plan = a.p;
  const Kv8Plan& p = a.p;
  for (const int32_t* x : {a.slots, a.lens, a.ntok}) sink += touch(x, sizeof(int32_t) * p.n);
  if (a.lens_out) std::memset(a.lens_out, 1, sizeof(int32_t) * p.n);
  // each array with a value of its own, so that two of them on one place are seen
  struct Part { void* at; size_t words; } parts[] = {
      {p.table, (size_t)p.num_slots * p.max_pages}, {p.owned, (size_t)p.num_slots},
      {p.free_pages, (size_t)p.num_pages}, {p.free_count, 1}, {p.mark, (size_t)p.num_slots},
      {p.status, 1}, {p.cu, (size_t)kKv8Rows + 1}, {p.pos, (size_t)p.T}, {p.map, (size_t)p.T},
      {p.tok_row, (size_t)p.T}, {p.rows, (size_t)4 * kKv8Rows}, {p.used, 2},
      {p.blocks, (size_t)kKv8Rows + 1}, {p.tiles, (size_t)kKv8Rows}};
  int value = 1;
  for (const Part& x : parts) std::memset(x.at, value++, 4 * x.words);
  value = 1;
  for (const Part& x : parts) {
    for (size_t i = 0; i < 4 * x.words; ++i)
      if (static_cast<unsigned char*>(x.at)[i] != value) return hipErrorInvalidValue;
    ++value;
  }
  return hipSuccess;
}

hipError_t launch_kv8_append(const Kv8AppendArgs& a) {
  ++gdn_fake::append_calls;
  tables(a.p);
  rows(a.k, a.p.T, a.ks, a.p.D, a.p.Hkv, a.p.D, 2);
  rows(a.v, a.p.T, a.vs, a.p.D, a.p.Hkv, a.p.D, 2);
  pages(a.p, a.pages, a.exps);
  return hipSuccess;
}

hipError_t launch_kv8_gather(const Kv8GatherArgs& a) {
  ++gdn_fake::gather_calls;
  sink += touch(a.map, sizeof(int32_t) * a.m);
  pages(a.p, a.pages, a.exps);
  if (a.k_out) rows(a.k_out, a.m, a.ks, a.p.D, a.p.Hkv, a.p.D, 2, 3);
  if (a.v_out) rows(a.v_out, a.m, a.vs, a.p.D, a.p.Hkv, a.p.D, 2, 4);
  return hipSuccess;
}

size_t kv8_attn_workspace_bytes(const gdn_kv8_desc& d) { return (size_t)64 * d.head_dim; }

hipError_t launch_kv8_attn(const Kv8AttnArgs& a) {
  ++gdn_fake::attn_calls;
  gdn_fake::attn8 = a;
  const Kv8Plan& p = a.p;
  tables(p);
  pages(p, a.pages, a.exps);
  rows(a.q, p.T, a.qs, a.qhs, p.Hq, p.D, 2);
  if (a.gate) rows(a.gate, p.T, a.gs, a.ghs, p.Hq, p.D, 2);
  if (a.slopes) sink += touch(a.slopes, sizeof(float) * p.Hq);
  if (a.prefix) sink += touch(a.prefix, sizeof(int32_t) * p.n);
  std::memset(a.workspace, 5, (size_t)64 * p.D);
  rows(a.out, p.T, a.os, a.ohs, p.Hq, p.D, 2, 6);
  return hipSuccess;
}

hipError_t launch_rope(const RopeArgs& a) {
  ++gdn_fake::rope_calls;
  sink += touch(a.turns, sizeof(double) * (a.rot / 2)) + touch(a.pos, sizeof(int32_t) * a.T);
  for (const gdn_rope_rows& r : {a.q, a.k}) {
    if (r.heads == 0) continue;
    rows(r.in, a.T, r.in_stride, r.in_head_stride, r.heads, a.D, a.f32 ? 4 : 2);
    if (r.norm_w) sink += touch(r.norm_w, sizeof(uint16_t) * a.D);
    rows(r.out, a.T, r.out_stride, r.out_head_stride, r.heads, a.D, a.f32 ? 4 : 2, 7);
  }
  return hipSuccess;
}

}  // namespace gdn
