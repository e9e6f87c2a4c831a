// gdn_kv8.cpp -- C ABI of the 8-bit paged KV cache that is planned on the GPU and of the
// rotary positions: argument checks, the lifetime of the device arrays, launches.
// See include/gdn.h for the contract.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <memory>
#include <new>
#include <stdexcept>
#include <vector>

#include "gdn.h"
#include "gdn_common.h"

namespace {

gdn_status kfail(gdn_status code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return gdn::set_error(code, buf);
}

gdn_status hip_fail(hipError_t e, const char* what) {
  return kfail(GDN_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

// Makes the cache's device current for the duration of a call.
class DeviceScope {
 public:
  explicit DeviceScope(int dev) {
    if (hipGetDevice(&prev_) != hipSuccess) prev_ = -1;
    if (prev_ != dev) ok_ = hipSetDevice(dev) == hipSuccess;
  }
  ~DeviceScope() {
    int cur = -1;
    if (ok_ && prev_ >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev_)
      (void)hipSetDevice(prev_);
  }
  bool ok() const { return ok_; }

 private:
  int prev_ = -1;
  bool ok_ = true;
};

constexpr int kPageTokens = 64;

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Rows of `heads` heads of `dim` elements, tokens `stride` and heads `head_stride` apart,
// the heads inside a token's row or the tokens inside a head's plane; every head starts
// at a multiple of `unit` elements. With `tokens` (an output's) no plane runs into the next.
bool rows_ok(const void* p, int64_t stride, int64_t head_stride, int heads, int dim, int unit,
             int elem, int64_t tokens = 1) {
  if (!aligned(p, (uintptr_t)unit * elem > 16 ? 16 : (uintptr_t)unit * elem) ||
      stride % unit != 0 || stride < dim)
    return false;
  if (heads <= 1) return true;
  return head_stride % unit == 0 && head_stride >= dim &&
         ((head_stride >= stride && head_stride >= (tokens - 1) * stride + dim) ||
          stride >= (heads - 1) * head_stride + dim);
}

// Rows of `heads` heads side by side, which do not run into the next row. A single row's stride
// does not matter.
bool packed_rows_ok(const void* p, int64_t stride, int heads, int dim, int64_t rows) {
  return aligned(p, 16) && (rows <= 1 || (stride % 8 == 0 && stride >= (int64_t)heads * dim));
}

}  // namespace

struct gdn_kv8 {
  gdn_kv8_desc d{};
  std::vector<uint8_t*> pages;  // per layer [num_pages][2][Hkv][64 * D]
  std::vector<int32_t*> exps;   // per layer [num_pages][2][Hkv]
  int32_t* ints = nullptr;      // the tables and the plan, one allocation
  void* workspace = nullptr;
  gdn::Kv8Plan p{};
  bool planned = false;
};

struct gdn_rope {
  gdn_rope_desc d{};
  int device = 0;
  float mag = 1.0f;
  double* turns = nullptr;  // [rotary_dim / 2] turns of a pair per position
};

namespace {

void kv8_free(gdn_kv8* kv) {
  if (!kv) return;
  for (uint8_t* p : kv->pages)
    if (p) (void)hipFree(p);
  for (int32_t* p : kv->exps)
    if (p) (void)hipFree(p);
  if (kv->ints) (void)hipFree(kv->ints);
  if (kv->workspace) (void)hipFree(kv->workspace);
  delete kv;
}

gdn_status check_layer(const gdn_kv8* kv, int32_t layer, const char* what) {
  if (!kv) return kfail(GDN_ERR_INVALID, "%s: NULL cache", what);
  if (layer < 0 || layer >= kv->d.num_layers)
    return kfail(GDN_ERR_INVALID, "%s: layer %d outside [0, %d)", what, layer, kv->d.num_layers);
  return GDN_OK;
}

}  // namespace

extern "C" {

gdn_status gdn_kv8_create(const gdn_kv8_desc* desc, gdn_kv8** out) try {
  if (!desc || !out) return kfail(GDN_ERR_INVALID, "gdn_kv8_create: desc/out is NULL");
  *out = nullptr;
  const gdn_kv8_desc& d = *desc;
  if (d.num_layers < 1 || d.num_slots < 1 || d.num_pages < 1 || d.max_pages_per_slot < 1 ||
      d.num_q_heads < 1 || d.num_kv_heads < 1 || d.max_step_tokens < 1)
    return kfail(GDN_ERR_INVALID, "gdn_kv8_create: sizes must be >= 1");
  if (d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 256)
    return kfail(GDN_ERR_UNSUPPORTED, "gdn_kv8_create: head_dim %d (64, 128 or 256)", d.head_dim);
  if (d.num_q_heads % d.num_kv_heads != 0 || d.num_q_heads / d.num_kv_heads > 16 ||
      d.num_kv_heads > 256)
    return kfail(GDN_ERR_UNSUPPORTED, "gdn_kv8_create: %d query heads on %d kv heads (1 to 16 for "
                 "each, at most 256 kv heads)", d.num_q_heads, d.num_kv_heads);
  if (d.num_slots > gdn::kKv8Rows || d.max_step_tokens > 262144 || d.num_pages > 1 << 24 ||
      d.max_pages_per_slot > 1 << 24 ||
      (int64_t)d.num_slots * d.max_pages_per_slot > (int64_t)1 << 30)
    return kfail(GDN_ERR_UNSUPPORTED, "gdn_kv8_create: %d slots (at most %d), %d step tokens "
                 "(262144), %d pages and %d of a slot (16777216 each, slots times it 2^30)",
                 d.num_slots, gdn::kKv8Rows, d.max_step_tokens, d.num_pages, d.max_pages_per_slot);
  DeviceScope dev(d.device);
  if (d.device < 0 || !dev.ok()) {
    (void)hipGetLastError();
    return kfail(GDN_ERR_INVALID, "gdn_kv8_create: no device %d", d.device);
  }
  std::unique_ptr<gdn_kv8, void (*)(gdn_kv8*)> held(new gdn_kv8, kv8_free);
  gdn_kv8* const kv = held.get();
  kv->d = d;
  kv->pages.reserve(d.num_layers);
  kv->exps.reserve(d.num_layers);
  const size_t page_bytes = (size_t)2 * d.num_kv_heads * kPageTokens * d.head_dim;
  const size_t heads = (size_t)2 * d.num_kv_heads * d.num_pages;
  const size_t table = (size_t)d.num_slots * d.max_pages_per_slot;
  const int R = gdn::kKv8Rows;
  const size_t words = table + 2 * (size_t)d.num_slots + d.num_pages + 4 + 7 * (size_t)(R + 1) +
                       3 * (size_t)d.max_step_tokens;
  const size_t ws = gdn::kv8_attn_workspace_bytes(d);
  bool ok = true;
  for (int l = 0; l < d.num_layers && ok; ++l) {
    uint8_t* p = nullptr;
    int32_t* e = nullptr;
    ok = hipMalloc(&p, page_bytes * d.num_pages) == hipSuccess;
    kv->pages.push_back(p);
    ok = ok && hipMalloc(&e, sizeof(int32_t) * heads) == hipSuccess;
    kv->exps.push_back(e);
    // positions that were never appended read as zeros
    ok = ok && hipMemset(p, 0, page_bytes * d.num_pages) == hipSuccess &&
         hipMemset(e, 0, sizeof(int32_t) * heads) == hipSuccess;
  }
  ok = ok && hipMalloc(&kv->ints, sizeof(int32_t) * words) == hipSuccess &&
       (ws == 0 || hipMalloc(&kv->workspace, ws) == hipSuccess);
  if (ok) {
    gdn::Kv8Plan& p = kv->p;
    p.num_slots = d.num_slots;
    p.num_pages = d.num_pages;
    p.max_pages = d.max_pages_per_slot;
    p.Hq = d.num_q_heads;
    p.Hkv = d.num_kv_heads;
    p.D = d.head_dim;
    int32_t* at = kv->ints;
    auto take = [&](size_t n) {
      int32_t* r = at;
      at += n;
      return r;
    };
    p.rows = reinterpret_cast<gdn::Kv8Row*>(take(4 * (size_t)R));  // 16-byte aligned
    p.table = take(table);
    p.owned = take(d.num_slots);
    p.mark = take(d.num_slots);
    p.free_pages = take(d.num_pages);
    p.free_count = take(1);
    p.used = take(2);
    p.status = reinterpret_cast<uint32_t*>(take(1));
    p.cu = take(R + 1);
    p.blocks = take(R + 1);
    p.tiles = take(R + 1);
    p.pos = take(d.max_step_tokens);
    p.map = take(d.max_step_tokens);
    p.tok_row = take(d.max_step_tokens);
    std::vector<int32_t> init(d.num_pages);
    for (int i = 0; i < d.num_pages; ++i) init[i] = d.num_pages - 1 - i;  // pop lowest first
    const std::vector<int32_t> mark(d.num_slots, INT_MAX), behind(R + 1, INT_MAX);
    ok = hipMemset(kv->ints, 0, sizeof(int32_t) * words) == hipSuccess &&
         hipMemset(p.table, 0xff, sizeof(int32_t) * table) == hipSuccess &&
         hipMemcpy(p.blocks, behind.data(), sizeof(int32_t) * (R + 1), hipMemcpyHostToDevice) ==
             hipSuccess &&
         hipMemcpy(p.free_pages, init.data(), sizeof(int32_t) * d.num_pages,
                   hipMemcpyHostToDevice) == hipSuccess &&
         hipMemcpy(p.mark, mark.data(), sizeof(int32_t) * d.num_slots, hipMemcpyHostToDevice) ==
             hipSuccess &&
         hipMemcpy(p.free_count, &d.num_pages, sizeof(int32_t), hipMemcpyHostToDevice) ==
             hipSuccess &&
         // other streams than the null stream may use the cache from here on
         hipDeviceSynchronize() == hipSuccess;
  }
  if (!ok) {
    (void)hipGetLastError();
    return kfail(GDN_ERR_OOM, "gdn_kv8_create: %d layers x %d pages of %zu bytes, workspace of %zu",
                 d.num_layers, d.num_pages, page_bytes, ws);
  }
  *out = held.release();
  return GDN_OK;
} catch (const std::bad_alloc&) {
  return kfail(GDN_ERR_OOM, "gdn_kv8_create: host memory");
} catch (const std::length_error&) {
  return kfail(GDN_ERR_OOM, "gdn_kv8_create: host memory");
}

gdn_status gdn_kv8_destroy(gdn_kv8* kv) {
  if (!kv) return GDN_OK;
  DeviceScope dev(kv->d.device);
  kv8_free(kv);
  return GDN_OK;
}

gdn_status gdn_kv8_describe(const gdn_kv8* kv, gdn_kv8_desc* desc) {
  if (!kv || !desc) return kfail(GDN_ERR_INVALID, "gdn_kv8_describe: NULL argument");
  *desc = kv->d;
  return GDN_OK;
}

gdn_status gdn_kv8_views(const gdn_kv8* kv, gdn_kv8_view* view) {
  if (!kv || !view) return kfail(GDN_ERR_INVALID, "gdn_kv8_views: NULL argument");
  const gdn::Kv8Plan& p = kv->p;
  *view = gdn_kv8_view{p.table, p.owned, p.free_pages, p.free_count, p.cu, p.pos, p.map};
  return GDN_OK;
}

gdn_status gdn_kv8_check(gdn_kv8* kv, void* stream, uint32_t* flags) {
  if (!kv || !flags) return kfail(GDN_ERR_INVALID, "gdn_kv8_check: NULL argument");
  DeviceScope dev(kv->d.device);
  hipError_t e = hipStreamSynchronize(static_cast<hipStream_t>(stream));
  uint32_t v = 0;
  if (e == hipSuccess) e = hipMemcpy(&v, kv->p.status, sizeof(v), hipMemcpyDeviceToHost);
  if (e == hipSuccess) e = hipMemset(kv->p.status, 0, sizeof(v));
  if (e == hipSuccess) e = hipDeviceSynchronize();
  if (e != hipSuccess) return hip_fail(e, "gdn_kv8_check");
  *flags = v;
  return GDN_OK;
}

gdn_status gdn_kv8_step(gdn_kv8* kv, int32_t n, const int32_t* slots, const int32_t* lens,
                        const int32_t* ntok, int32_t* lens_out, int32_t max_tokens,
                        int32_t max_row_tokens, void* stream) {
  if (!kv) return kfail(GDN_ERR_INVALID, "gdn_kv8_step: NULL cache");
  if (!slots || !lens || !ntok) return kfail(GDN_ERR_INVALID, "gdn_kv8_step: NULL array");
  for (const int32_t* p : {slots, lens, ntok, (const int32_t*)lens_out})
    if (!aligned(p, 4)) return kfail(GDN_ERR_INVALID, "gdn_kv8_step: an array is not aligned");
  if (n < 1 || n > gdn::kKv8Rows)
    return kfail(GDN_ERR_INVALID, "gdn_kv8_step: n = %d outside [1, %d]", n, gdn::kKv8Rows);
  if (max_tokens < 0 || max_tokens > kv->d.max_step_tokens)
    return kfail(GDN_ERR_INVALID, "gdn_kv8_step: max_tokens = %d outside [0, %d]", max_tokens,
                 kv->d.max_step_tokens);
  if (max_row_tokens < 0 || max_row_tokens > max_tokens)
    return kfail(GDN_ERR_INVALID, "gdn_kv8_step: max_row_tokens = %d outside [0, %d]",
                 max_row_tokens, max_tokens);
  DeviceScope dev(kv->d.device);
  gdn::Kv8StepArgs a{};
  a.p = kv->p;
  a.p.n = n;
  a.p.T = max_tokens;
  a.p.max_row = max_row_tokens ? max_row_tokens : max_tokens;
  a.slots = slots;
  a.lens = lens;
  a.ntok = ntok;
  a.lens_out = lens_out;
  a.stream = static_cast<hipStream_t>(stream);
  const hipError_t e = gdn::launch_kv8_step(a);
  if (e != hipSuccess) return hip_fail(e, "gdn_kv8_step launch");
  kv->p = a.p;
  kv->planned = true;
  return GDN_OK;
}

gdn_status gdn_kv8_append(gdn_kv8* kv, int32_t layer, const uint16_t* k, int64_t k_stride,
                          const uint16_t* v, int64_t v_stride, void* stream) {
  const gdn_status st = check_layer(kv, layer, "gdn_kv8_append");
  if (st != GDN_OK) return st;
  if (!kv->planned) return kfail(GDN_ERR_INVALID, "gdn_kv8_append: no step planned (gdn_kv8_step)");
  if (kv->p.T == 0) return GDN_OK;
  if (!k || !v) return kfail(GDN_ERR_INVALID, "gdn_kv8_append: NULL tensor pointer");
  const int D = kv->d.head_dim, H = kv->d.num_kv_heads;
  if (!packed_rows_ok(k, k_stride, H, D, kv->p.T) || !packed_rows_ok(v, v_stride, H, D, kv->p.T))
    return kfail(GDN_ERR_INVALID, "gdn_kv8_append: k and v need 16-byte alignment and row strides "
                 ">= %d that are multiples of 8 (got %lld, %lld)", H * D, (long long)k_stride,
                 (long long)v_stride);
  DeviceScope dev(kv->d.device);
  gdn::Kv8AppendArgs a{};
  a.p = kv->p;
  a.pages = kv->pages[layer];
  a.exps = kv->exps[layer];
  a.k = k;
  a.ks = k_stride;
  a.v = v;
  a.vs = v_stride;
  a.stream = static_cast<hipStream_t>(stream);
  const hipError_t e = gdn::launch_kv8_append(a);
  return e == hipSuccess ? GDN_OK : hip_fail(e, "gdn_kv8_append launch");
}

gdn_status gdn_kv8_gather(gdn_kv8* kv, int32_t layer, int32_t m, const int32_t* map,
                          uint16_t* k_out, int64_t k_stride, uint16_t* v_out, int64_t v_stride,
                          void* stream) {
  const gdn_status st = check_layer(kv, layer, "gdn_kv8_gather");
  if (st != GDN_OK) return st;
  if (m < 0 || m > 1 << 24) return kfail(GDN_ERR_INVALID, "gdn_kv8_gather: m = %d", m);
  if (m == 0) return GDN_OK;
  if (!map || !aligned(map, 4) || (!k_out && !v_out))
    return kfail(GDN_ERR_INVALID, "gdn_kv8_gather: NULL or misaligned array");
  const int D = kv->d.head_dim, H = kv->d.num_kv_heads;
  if ((k_out && !packed_rows_ok(k_out, k_stride, H, D, m)) ||
      (v_out && !packed_rows_ok(v_out, v_stride, H, D, m)))
    return kfail(GDN_ERR_INVALID, "gdn_kv8_gather: outputs need 16-byte alignment and row strides "
                 ">= %d that are multiples of 8 (got %lld, %lld)", H * D, (long long)k_stride,
                 (long long)v_stride);
  DeviceScope dev(kv->d.device);
  gdn::Kv8GatherArgs a{};
  a.p = kv->p;
  a.pages = kv->pages[layer];
  a.exps = kv->exps[layer];
  a.m = m;
  a.map = map;
  a.k_out = k_out;
  a.ks = k_stride;
  a.v_out = v_out;
  a.vs = v_stride;
  a.stream = static_cast<hipStream_t>(stream);
  const hipError_t e = gdn::launch_kv8_gather(a);
  return e == hipSuccess ? GDN_OK : hip_fail(e, "gdn_kv8_gather launch");
}

gdn_status gdn_kv8_attention(gdn_kv8* kv, int32_t layer, const gdn_kv8_attn_desc* desc,
                             const uint16_t* q, int64_t q_stride, int64_t q_head_stride,
                             const float* slopes, const int32_t* prefix, const uint16_t* gate,
                             int64_t gate_stride, int64_t gate_head_stride, uint16_t* out,
                             int64_t out_stride, int64_t out_head_stride, void* stream) {
  const gdn_status st = check_layer(kv, layer, "gdn_kv8_attention");
  if (st != GDN_OK) return st;
  if (!desc) return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: NULL descriptor");
  if (!kv->planned)
    return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: no step planned (gdn_kv8_step)");
  if (!std::isfinite(desc->scale) || !std::isfinite(desc->softcap) || desc->softcap < 0.0f ||
      (desc->softcap != 0.0f && (desc->softcap < 1e-30f || desc->softcap > 1e30f)) ||
      desc->window < 0)
    return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: scale %g, softcap %g, window %d",
                 (double)desc->scale, (double)desc->softcap, desc->window);
  if (kv->p.T == 0) return GDN_OK;
  if (!q || !out) return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: NULL tensor pointer");
  const int D = kv->d.head_dim, H = kv->d.num_q_heads;
  if (!rows_ok(q, q_stride, q_head_stride, H, D, 8, 2))
    return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: q needs 16-byte alignment and strides that "
                 "hold %d heads of %d in multiples of 8", H, D);
  if (gate && !rows_ok(gate, gate_stride, gate_head_stride, H, D, 8, 2))
    return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: gate needs 16-byte alignment and strides "
                 "that hold %d heads of %d in multiples of 8", H, D);
  if (!rows_ok(out, out_stride, out_head_stride, H, D, 4, 2, kv->p.T))
    return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: out needs 8-byte alignment and strides that "
                 "hold %d heads of %d in multiples of 4", H, D);
  if (!aligned(slopes, 4) || !aligned(prefix, 4))
    return kfail(GDN_ERR_INVALID, "gdn_kv8_attention: slopes or prefix is not aligned");
  DeviceScope dev(kv->d.device);
  gdn::Kv8AttnArgs a{};
  a.p = kv->p;
  a.pages = kv->pages[layer];
  a.exps = kv->exps[layer];
  a.scale = desc->scale != 0.0f ? desc->scale : 1.0f / std::sqrt((float)D);
  a.softcap = desc->softcap;
  a.window = desc->window;
  a.q = q;
  a.qs = q_stride;
  a.qhs = q_head_stride;
  a.slopes = slopes;
  a.prefix = prefix;
  a.gate = gate;
  a.gs = gate_stride;
  a.ghs = gate_head_stride;
  a.out = out;
  a.os = out_stride;
  a.ohs = out_head_stride;
  a.workspace = kv->workspace;
  a.stream = static_cast<hipStream_t>(stream);
  const hipError_t e = gdn::launch_kv8_attn(a);
  return e == hipSuccess ? GDN_OK : hip_fail(e, "gdn_kv8_attention launch");
}

gdn_status gdn_rope_create(const gdn_rope_desc* desc, int32_t device, gdn_rope** out) try {
  if (!desc || !out) return kfail(GDN_ERR_INVALID, "gdn_rope_create: desc/out is NULL");
  *out = nullptr;
  const gdn_rope_desc& d = *desc;
  if (d.head_dim < 8 || d.head_dim > 512 || d.head_dim % 8 != 0)
    return kfail(GDN_ERR_UNSUPPORTED, "gdn_rope_create: head_dim %d not a multiple of 8 in [8, 512]",
                 d.head_dim);
  if (d.rotary_dim < 0 || d.rotary_dim > d.head_dim || d.rotary_dim % 2 != 0)
    return kfail(GDN_ERR_INVALID, "gdn_rope_create: rotary_dim %d", d.rotary_dim);
  if (d.scaling < GDN_ROPE_NONE || d.scaling > GDN_ROPE_BANDS)
    return kfail(GDN_ERR_INVALID, "gdn_rope_create: scaling %d", d.scaling);
  if (!std::isfinite(d.base) || !(d.base > 1.0f) || !std::isfinite(d.factor) ||
      !(d.factor > 0.0f) || !std::isfinite(d.magnitude))
    return kfail(GDN_ERR_INVALID, "gdn_rope_create: base, factor or magnitude");
  if (d.scaling >= GDN_ROPE_YARN &&
      (!std::isfinite(d.original) || !(d.original > 0.0f) || !std::isfinite(d.fast) ||
       !(d.slow > 0.0f) || !(d.fast > d.slow)))
    return kfail(GDN_ERR_INVALID, "gdn_rope_create: original, fast or slow");
  DeviceScope dev(device);
  if (device < 0 || !dev.ok()) {
    (void)hipGetLastError();
    return kfail(GDN_ERR_INVALID, "gdn_rope_create: no device %d", device);
  }
  std::unique_ptr<gdn_rope> held(new gdn_rope);
  gdn_rope* const r = held.get();
  r->d = d;
  r->device = device;
  const double pi = 3.14159265358979323846, rot = d.rotary_dim, base = d.base, f = d.factor;
  r->mag = d.magnitude != 0.0f ? d.magnitude
           : d.scaling == GDN_ROPE_YARN ? (float)(0.1 * std::log(f) + 1.0) : 1.0f;
  const int half = d.rotary_dim / 2;
  std::vector<double> turns(std::max(half, 1));
  auto dim_of = [&](double b) {
    return rot * std::log(d.original / (2.0 * pi * b)) / (2.0 * std::log(base));
  };
  const double lo = std::max(std::floor(dim_of(d.fast)), 0.0);
  const double hi = std::min(std::ceil(dim_of(d.slow)), rot - 1.0);
  for (int i = 0; i < half; ++i) {
    double w = std::pow(base, -2.0 * i / rot);
    if (d.scaling == GDN_ROPE_LINEAR) w /= f;
    if (d.scaling == GDN_ROPE_YARN) {
      const double s = std::min(std::max((i - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
      w = w / f * s + w * (1.0 - s);
    }
    if (d.scaling == GDN_ROPE_BANDS) {
      const double t = d.original * w / (2.0 * pi);
      const double k = std::min(std::max((t - d.slow) / ((double)d.fast - d.slow), 0.0), 1.0);
      w = w / f * (1.0 - k) + w * k;
    }
    turns[i] = w / (2.0 * pi);
  }
  if (hipMalloc(&r->turns, sizeof(double) * turns.size()) != hipSuccess ||
      hipMemcpy(r->turns, turns.data(), sizeof(double) * turns.size(), hipMemcpyHostToDevice) !=
          hipSuccess ||
      hipDeviceSynchronize() != hipSuccess) {
    (void)hipGetLastError();
    if (r->turns) (void)hipFree(r->turns);
    return kfail(GDN_ERR_OOM, "gdn_rope_create: %zu bytes", sizeof(double) * turns.size());
  }
  *out = held.release();
  return GDN_OK;
} catch (const std::bad_alloc&) {
  return kfail(GDN_ERR_OOM, "gdn_rope_create: host memory");
}

gdn_status gdn_rope_destroy(gdn_rope* rope) {
  if (!rope) return GDN_OK;
  DeviceScope dev(rope->device);
  if (rope->turns) (void)hipFree(rope->turns);
  delete rope;
  return GDN_OK;
}

gdn_status gdn_rope_forward(const gdn_rope* rope, int32_t T, const int32_t* pos,
                            const gdn_rope_rows* q, const gdn_rope_rows* k, int32_t f32, float eps,
                            int32_t inverse, void* stream) {
  if (!rope) return kfail(GDN_ERR_INVALID, "gdn_rope_forward: NULL handle");
  if (!q) return kfail(GDN_ERR_INVALID, "gdn_rope_forward: q is NULL");
  if (T < 0 || T > 1 << 24) return kfail(GDN_ERR_INVALID, "gdn_rope_forward: T = %d", T);
  if (!(eps >= 0.0f)) return kfail(GDN_ERR_INVALID, "gdn_rope_forward: eps must be >= 0");
  if (T == 0) return GDN_OK;
  if (!pos || !aligned(pos, 4))
    return kfail(GDN_ERR_INVALID, "gdn_rope_forward: pos is NULL or not aligned");
  const int D = rope->d.head_dim, elem = f32 ? 4 : 2;
  const gdn_rope_rows none{};
  for (const gdn_rope_rows* r : {q, k}) {
    if (!r) continue;
    const char* name = r == q ? "q" : "k";
    if (r->heads < (r == q ? 1 : 0) || r->heads > 4096)
      return kfail(GDN_ERR_INVALID, "gdn_rope_forward: %s has %d heads", name, r->heads);
    if (r->heads == 0) continue;
    if (!r->in || !r->out || !rows_ok(r->in, r->in_stride, r->in_head_stride, r->heads, D, 8, elem) ||
        !rows_ok(r->out, r->out_stride, r->out_head_stride, r->heads, D, 8, elem, T) ||
        !aligned(r->norm_w, 16))
      return kfail(GDN_ERR_INVALID, "gdn_rope_forward: %s needs 16-byte alignment and strides that "
                   "hold %d heads of %d in multiples of 8", name, r->heads, D);
    if (inverse && r->norm_w)
      return kfail(GDN_ERR_INVALID, "gdn_rope_forward: the inverse turns without norm weights");
    if (r->in == r->out &&
        (r->in_stride != r->out_stride || r->in_head_stride != r->out_head_stride))
      return kfail(GDN_ERR_INVALID, "gdn_rope_forward: %s turned in place keeps its strides", name);
  }
  DeviceScope dev(rope->device);
  gdn::RopeArgs a{};
  a.D = D;
  a.rot = rope->d.rotary_dim;
  a.interleaved = rope->d.interleaved != 0;
  a.f32 = f32 != 0;
  a.inverse = inverse != 0;
  a.mag = rope->mag;
  a.eps = eps;
  a.turns = rope->turns;
  a.T = T;
  a.pos = pos;
  a.q = *q;
  a.k = k ? *k : none;
  a.stream = static_cast<hipStream_t>(stream);
  const hipError_t e = gdn::launch_rope(a);
  return e == hipSuccess ? GDN_OK : hip_fail(e, "gdn_rope_forward launch");
}

}  // extern "C"
