// gdn_moe.cpp -- C ABI of the decoder layer's sparse MLP half: argument checks
// and launches of the router and the block norm, and the lifetime of the
// experts' packed weights. See include/gdn.h for the contract.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <new>

#include "gdn.h"
#include "gdn_common.h"

namespace {

gdn_status mfail(gdn_status code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return gdn::set_error(code, buf);
}

gdn_status hip_fail(hipError_t e, const char* what) {
  return mfail(GDN_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

// Makes the layer's device current for the duration of a call.
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

// Rows of one launch of the kernels with a work-group or a wave a row: a grid
// holds less than 2^32 threads, of which a row takes up to 512.
constexpr int64_t kRowsOfLaunch = 1 << 22;

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

struct gdn_moe {
  int hidden = 0, inner = 0, experts = 0, device = 0;
  void* base = nullptr;  // one allocation holds the packed arrays
  void* w1 = nullptr;
  uint32_t* sb1 = nullptr;
  void* w2 = nullptr;
  uint32_t* sb2 = nullptr;
  float* bound = nullptr;
};

namespace {

void moe_release(gdn_moe* m) {
  if (!m) return;
  if (m->base) (void)hipFree(m->base);
  delete m;
}

}  // namespace

namespace {

// What an executor's MLP halves share: the rows between their steps.
struct ExecMoeBuffers {
  uint16_t* logits = nullptr;
  int32_t* ids = nullptr;
  float* weights = nullptr;
  void* workspace = nullptr;
  size_t workspace_bytes = 0;
  ~ExecMoeBuffers() {
    for (void* p : {(void*)logits, (void*)ids, (void*)weights, workspace})
      if (p) (void)hipFree(p);
  }
};

struct ExecMoe {
  const gdn_qlinear* gate = nullptr;
  int64_t gate_cols = 0;
  gdn_moe_route_desc route{};
  const float* bias = nullptr;
  const gdn_moe* moe = nullptr;
  std::shared_ptr<ExecMoeBuffers> buf;
};

gdn_status run_exec_moe(void* ctx, const uint16_t* hn, int n, uint16_t* out, hipStream_t s) {
  const ExecMoe& m = *static_cast<const ExecMoe*>(ctx);
  const int k = m.route.top_k + m.route.num_shared;
  gdn_status st = gdn_qlinear_forward(m.gate, hn, m.moe->hidden, n, m.buf->logits, m.gate_cols, s);
  if (st != GDN_OK) return st;
  st = gdn_moe_route(&m.route, m.buf->logits, m.gate_cols, n, m.bias, m.buf->ids, m.buf->weights, s);
  if (st != GDN_OK) return st;
  return gdn_moe_forward(m.moe, hn, m.moe->hidden, n, k, m.buf->ids, m.buf->weights, out,
                         m.moe->hidden, m.buf->workspace, m.buf->workspace_bytes, s);
}

}  // namespace

extern "C" {

gdn_status gdn_moe_route(const gdn_moe_route_desc* desc, const void* logits,
                         int64_t logits_stride, int32_t T, const float* bias, int32_t* ids,
                         float* weights, void* stream) {
  if (!desc) return mfail(GDN_ERR_INVALID, "gdn_moe_route: NULL descriptor");
  const gdn_moe_route_desc& d = *desc;
  if (d.num_experts < 1 || d.num_experts > 1024)
    return mfail(GDN_ERR_UNSUPPORTED, "gdn_moe_route: num_experts = %d outside [1, 1024]",
                 d.num_experts);
  if (d.top_k < 1 || d.top_k > 32 || d.top_k > d.num_experts)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: top_k = %d outside [1, min(%d, 32)]", d.top_k,
                 d.num_experts);
  if (d.score != GDN_MOE_SOFTMAX && d.score != GDN_MOE_SIGMOID)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: score = %d", d.score);
  if (d.num_groups < 1 || d.num_groups > 64 || d.num_experts % d.num_groups != 0)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: num_groups = %d must divide num_experts = %d "
                 "and be at most 64", d.num_groups, d.num_experts);
  if (d.top_groups < 1 || d.top_groups > d.num_groups)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: top_groups = %d outside [1, %d]", d.top_groups,
                 d.num_groups);
  if (d.group_top != 1 && d.group_top != 2)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: group_top = %d (1 or 2)", d.group_top);
  if (d.num_shared < 0 || d.num_shared > 8)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: num_shared = %d outside [0, 8]", d.num_shared);
  if (d.shared_gate && d.num_shared == 0)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: shared_gate without shared experts");
  if (!(d.scale - d.scale == 0.0f))
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: scale must be finite");
  if (T < 0) return mfail(GDN_ERR_INVALID, "gdn_moe_route: T = %d < 0", T);
  if (T == 0) return GDN_OK;
  if (!logits || !ids || !weights)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: NULL tensor pointer");
  const int cols = d.num_experts + (d.shared_gate ? 1 : 0);
  if (logits_stride < cols)
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: logits_stride %lld < %d columns",
                 (long long)logits_stride, cols);
  if (!aligned(logits, d.logits_f32 ? 4 : 2) || !aligned(ids, 4) || !aligned(weights, 4) ||
      !aligned(bias, 4))
    return mfail(GDN_ERR_INVALID, "gdn_moe_route: tensors need their element's alignment");
  gdn::MoeRouteArgs a{};
  a.d = d;
  a.stride = logits_stride;
  a.bias = bias;
  a.stream = static_cast<hipStream_t>(stream);
  for (int64_t t = 0; t < T; t += kRowsOfLaunch) {
    a.T = (int)std::min<int64_t>(T - t, kRowsOfLaunch);
    a.logits = static_cast<const char*>(logits) + t * logits_stride * (d.logits_f32 ? 4 : 2);
    a.ids = ids + t * (d.top_k + d.num_shared);
    a.weights = weights + t * (d.top_k + d.num_shared);
    const hipError_t e = gdn::launch_moe_route(a);
    if (e != hipSuccess) return hip_fail(e, "gdn_moe_route launch");
  }
  return GDN_OK;
}

gdn_status gdn_moe_create(int32_t hidden, int32_t inner, int32_t nparts, const gdn_moe_part* parts,
                          int32_t group_size, int32_t bits, int32_t device, void* stream,
                          gdn_moe** out) {
  if (!out) return mfail(GDN_ERR_INVALID, "gdn_moe_create: out is NULL");
  *out = nullptr;
  if (bits != 4 || group_size != 64)
    return mfail(GDN_ERR_UNSUPPORTED, "gdn_moe_create: bits = %d, group_size = %d (need 4, 64)",
                 bits, group_size);
  for (int32_t v : {hidden, inner})
    if (v < 128 || v > 8192 || v % 128 != 0)
      return mfail(GDN_ERR_UNSUPPORTED, "gdn_moe_create: hidden = %d and inner = %d must be "
                   "multiples of 128 in [128, 8192]", hidden, inner);
  if (nparts < 1 || nparts > 64 || !parts)
    return mfail(GDN_ERR_INVALID, "gdn_moe_create: nparts = %d / NULL parts", nparts);
  int64_t experts = 0;
  for (int i = 0; i < nparts; ++i) {
    const gdn_moe_part& p = parts[i];
    if (p.experts < 1)
      return mfail(GDN_ERR_INVALID, "gdn_moe_create: part %d has %d experts", i, p.experts);
    for (const void* t : {(const void*)p.gate_w, (const void*)p.gate_scales,
                          (const void*)p.gate_biases, (const void*)p.up_w,
                          (const void*)p.up_scales, (const void*)p.up_biases,
                          (const void*)p.down_w, (const void*)p.down_scales,
                          (const void*)p.down_biases})
      if (!t || !aligned(t, 2))
        return mfail(GDN_ERR_INVALID, "gdn_moe_create: part %d has a NULL or misaligned tensor", i);
    if (!aligned(p.gate_w, 4) || !aligned(p.up_w, 4) || !aligned(p.down_w, 4))
      return mfail(GDN_ERR_INVALID, "gdn_moe_create: part %d has misaligned weights", i);
    experts += p.experts;
  }
  if (experts > 4096)
    return mfail(GDN_ERR_UNSUPPORTED, "gdn_moe_create: %lld experts > 4096", (long long)experts);
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || device < 0 || device >= ndev)
    return mfail(GDN_ERR_INVALID, "gdn_moe_create: device %d not present", device);
  DeviceScope scope(device);
  if (!scope.ok()) return mfail(GDN_ERR_HIP, "gdn_moe_create: hipSetDevice(%d) failed", device);

  gdn_moe* m = new (std::nothrow) gdn_moe;
  if (!m) return mfail(GDN_ERR_OOM, "gdn_moe_create: out of host memory");
  m->hidden = hidden;
  m->inner = inner;
  m->experts = (int)experts;
  m->device = device;
  // one expert's matrix product terms: words of 8 weights, {scale, bias} per 64
  const size_t terms = (size_t)hidden * inner;
  const size_t w = terms / 2 * experts, s = terms / 16 * experts;
  const size_t bytes = 3 * (w + s) + 12 * (size_t)experts;  // w, s multiples of 1024 bytes
  if (hipMalloc(&m->base, bytes) != hipSuccess) {
    (void)hipGetLastError();
    m->base = nullptr;
    moe_release(m);
    return mfail(GDN_ERR_OOM, "gdn_moe_create: hipMalloc of %zu bytes failed", bytes);
  }
  char* p = static_cast<char*>(m->base);
  m->w1 = p;
  m->w2 = p + 2 * w;
  m->sb1 = reinterpret_cast<uint32_t*>(p + 3 * w);
  m->sb2 = reinterpret_cast<uint32_t*>(p + 3 * w + 2 * s);
  m->bound = reinterpret_cast<float*>(p + 3 * (w + s));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = hipMemsetAsync(m->bound, 0, 12 * (size_t)experts, st);
  int64_t first = 0;
  for (int i = 0; i < nparts; ++i) {
    const gdn_moe_part& q = parts[i];
    gdn::MoePackArgs a{};
    a.experts = q.experts;
    a.stream = st;
    auto pack = [&](const uint32_t* wsrc, const uint16_t* ssrc, const uint16_t* bsrc, int n, int k,
                    int fmul, int fofs, void* wp, uint32_t* sb) {
      a.w = wsrc;
      a.s = ssrc;
      a.b = bsrc;
      a.n = n;
      a.k = k;
      a.fmul = fmul;
      a.fofs = fofs;
      a.frags = fmul * (n / 16);
      a.wp = static_cast<char*>(wp) + first * fmul * (terms / 2);
      a.sb = sb + first * fmul * (terms / 64);
      return gdn::launch_moe_pack(a);
    };
    // of the matrices packed last
    auto bound = [&](int which) {
      return gdn::launch_moe_bound(a, which == 2, m->bound + which * experts + first);
    };
    if (e == hipSuccess)
      e = pack(q.gate_w, q.gate_scales, q.gate_biases, inner, hidden, 2, 0, m->w1, m->sb1);
    if (e == hipSuccess) e = bound(0);
    if (e == hipSuccess)
      e = pack(q.up_w, q.up_scales, q.up_biases, inner, hidden, 2, 1, m->w1, m->sb1);
    if (e == hipSuccess) e = bound(1);
    if (e == hipSuccess)
      e = pack(q.down_w, q.down_scales, q.down_biases, hidden, inner, 1, 0, m->w2, m->sb2);
    if (e == hipSuccess) e = bound(2);
    if (e != hipSuccess) {
      (void)hipStreamSynchronize(st);
      moe_release(m);
      return hip_fail(e, "gdn_moe_create: pack");
    }
    first += q.experts;
  }
  e = hipStreamSynchronize(st);
  if (e != hipSuccess) {
    moe_release(m);
    return hip_fail(e, "gdn_moe_create: synchronize");
  }
  *out = m;
  return GDN_OK;
}

gdn_status gdn_moe_destroy(gdn_moe* m) {
  if (!m) return GDN_OK;
  DeviceScope scope(m->device);
  moe_release(m);
  return GDN_OK;
}

gdn_status gdn_moe_dims(const gdn_moe* m, int32_t* hidden, int32_t* inner, int32_t* experts) {
  if (!m) return mfail(GDN_ERR_INVALID, "gdn_moe_dims: NULL layer");
  if (hidden) *hidden = m->hidden;
  if (inner) *inner = m->inner;
  if (experts) *experts = m->experts;
  return GDN_OK;
}

gdn_status gdn_moe_workspace_bytes(const gdn_moe* m, int32_t T, int32_t k, size_t* bytes) {
  if (!m || !bytes) return mfail(GDN_ERR_INVALID, "gdn_moe_workspace_bytes: NULL argument");
  if (T < 0 || k < 1 || k > 64)
    return mfail(GDN_ERR_INVALID, "gdn_moe_workspace_bytes: T = %d < 0 or k = %d outside [1, 64]",
                 T, k);
  *bytes = gdn::moe_workspace_bytes(m->hidden, m->inner, m->experts, T, k);
  return GDN_OK;
}

gdn_status gdn_moe_forward(const gdn_moe* m, const uint16_t* x, int64_t x_stride, int32_t T,
                           int32_t k, const int32_t* ids, const float* weights, uint16_t* out,
                           int64_t out_stride, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (!m) return mfail(GDN_ERR_INVALID, "gdn_moe_forward: NULL layer");
  if (T < 0) return mfail(GDN_ERR_INVALID, "gdn_moe_forward: T = %d < 0", T);
  if (k < 1 || k > 64)
    return mfail(GDN_ERR_INVALID, "gdn_moe_forward: k = %d outside [1, 64]", k);
  if (T == 0) return GDN_OK;
  if (!x || !ids || !weights || !out || !workspace)
    return mfail(GDN_ERR_INVALID, "gdn_moe_forward: NULL tensor pointer");
  if (x_stride < m->hidden || x_stride % 8 != 0 || !aligned(x, 16))
    return mfail(GDN_ERR_INVALID, "gdn_moe_forward: x needs 16-byte alignment and a row stride >= "
                 "%d that is a multiple of 8 (got %lld)", m->hidden, (long long)x_stride);
  if (out_stride < m->hidden || out_stride % 4 != 0 || !aligned(out, 8))
    return mfail(GDN_ERR_INVALID, "gdn_moe_forward: out needs 8-byte alignment and a row stride "
                 ">= %d that is a multiple of 4 (got %lld)", m->hidden, (long long)out_stride);
  if (!aligned(ids, 4) || !aligned(weights, 4) || !aligned(workspace, 256))
    return mfail(GDN_ERR_INVALID, "gdn_moe_forward: ids and weights need 4-byte alignment, "
                 "workspace 256-byte alignment");
  const size_t need = gdn::moe_workspace_bytes(m->hidden, m->inner, m->experts, T, k);
  if (workspace_bytes < need)
    return mfail(GDN_ERR_INVALID, "gdn_moe_forward: workspace of %zu bytes, %zu needed",
                 workspace_bytes, need);
  DeviceScope scope(m->device);
  if (!scope.ok()) return mfail(GDN_ERR_HIP, "gdn_moe_forward: hipSetDevice(%d) failed", m->device);
  gdn::MoeArgs a{};
  a.hidden = m->hidden;
  a.inner = m->inner;
  a.experts = m->experts;
  a.w1 = m->w1;
  a.sb1 = m->sb1;
  a.w2 = m->w2;
  a.sb2 = m->sb2;
  a.bound = m->bound;
  a.xs = x_stride;
  a.k = k;
  a.os = out_stride;
  a.workspace = workspace;
  a.stream = static_cast<hipStream_t>(stream);
  const int pass = gdn::moe_pass_tokens(k, x_stride);
  for (int64_t t = 0; t < T; t += pass) {
    a.T = (int)(T - t < pass ? T - t : pass);
    a.x = x + t * x_stride;
    a.ids = ids + t * k;
    a.weights = weights + t * k;
    a.out = out + t * out_stride;
    const hipError_t e = gdn::launch_moe(a);
    if (e != hipSuccess) return hip_fail(e, "gdn_moe_forward launch");
  }
  return GDN_OK;
}

gdn_status gdn_exec_set_moe(gdn_exec* exec, int32_t n, const gdn_exec_moe* layers) try {
  if (!exec) return mfail(GDN_ERR_INVALID, "gdn_exec_set_moe: NULL executor");
  const gdn::ExecShape x = gdn::exec_shape(exec);
  if (x.held > 0 || x.pending)
    return mfail(GDN_ERR_INVALID, "gdn_exec_set_moe: the executor holds %zu sequences", x.held);
  if (n < 0 || n > x.depth || (n > 0 && !layers))
    return mfail(GDN_ERR_INVALID, "gdn_exec_set_moe: n = %d (a stack of %d layers) / NULL layers", n,
                 x.depth);
  std::vector<char> taken(x.depth, 0);
  std::vector<gdn::ExecMlp> halves(n);
  std::vector<std::shared_ptr<ExecMoe>> moes(n);
  int64_t cols = 0;
  int entries = 0;
  size_t workspace = 0;
  for (int i = 0; i < n; ++i) {
    const gdn_exec_moe& l = layers[i];
    if (l.position < 0 || l.position >= x.depth || taken[l.position])
      return mfail(GDN_ERR_INVALID, "gdn_exec_set_moe: half %d at position %d (distinct, < %d)", i,
                   l.position, x.depth);
    taken[l.position] = 1;
    if (!l.norm_w || !l.gate || !l.route || !l.moe || !aligned(l.norm_w, 16) || !aligned(l.bias, 4))
      return mfail(GDN_ERR_INVALID, "gdn_exec_set_moe: half %d has a NULL or misaligned weight", i);
    const gdn_moe_route_desc& r = *l.route;
    int32_t gk = 0, gn = 0;
    gdn_status st = gdn_qlinear_dims(l.gate, &gk, &gn);
    if (st != GDN_OK) return st;
    if (gk != x.hidden || l.moe->hidden != x.hidden || l.moe->device != x.device ||
        gn < r.num_experts + (r.shared_gate ? 1 : 0) || r.logits_f32 ||
        (int64_t)r.num_experts + r.num_shared != l.moe->experts)
      return mfail(GDN_ERR_INVALID, "gdn_exec_set_moe: half %d: gate %d -> %d, %d + %d experts "
                   "routed, layer of %d experts, hidden %d, device %d; executor hidden %d, device %d",
                   i, gk, gn, r.num_experts, r.num_shared, l.moe->experts, l.moe->hidden,
                   l.moe->device, x.hidden, x.device);
    st = gdn_moe_route(&r, nullptr, 0, 0, nullptr, nullptr, nullptr, nullptr);  // its descriptor
    if (st != GDN_OK) return st;
    auto m = std::make_shared<ExecMoe>();
    m->gate = l.gate;
    m->gate_cols = gn;
    m->route = r;
    m->bias = l.bias;
    m->moe = l.moe;
    moes[i] = m;
    const int k = r.top_k + r.num_shared;
    if (gn > cols) cols = gn;
    if (k > entries) entries = k;
    const size_t w = gdn::moe_workspace_bytes(x.hidden, l.moe->inner, l.moe->experts, x.rows, k);
    if (w > workspace) workspace = w;
    halves[i].position = l.position;
    halves[i].norm_w = l.norm_w;
    halves[i].run = run_exec_moe;
    halves[i].ctx = m;
  }
  if (n > 0) {
    DeviceScope scope(x.device);
    auto buf = std::make_shared<ExecMoeBuffers>();
    buf->workspace_bytes = workspace;
    if (hipMalloc(&buf->logits, (size_t)x.rows * cols * 2) != hipSuccess ||
        hipMalloc(&buf->ids, (size_t)x.rows * entries * 4) != hipSuccess ||
        hipMalloc(&buf->weights, (size_t)x.rows * entries * 4) != hipSuccess ||
        hipMalloc(&buf->workspace, workspace) != hipSuccess) {
      (void)hipGetLastError();
      return mfail(GDN_ERR_OOM, "gdn_exec_set_moe: buffers for %d rows (%zu bytes of workspace)",
                   x.rows, workspace);
    }
    for (auto& m : moes) m->buf = buf;
  }
  return gdn::exec_set_mlp(exec, std::move(halves));
} catch (const std::bad_alloc&) {
  return mfail(GDN_ERR_OOM, "gdn_exec_set_moe: out of host memory");
}

gdn_status gdn_block_norm(const gdn_block_norm_desc* desc, int32_t n, const void* h,
                          int64_t h_stride, const uint16_t* x, int64_t x_stride,
                          const uint16_t* post_w, const uint16_t* gate, int64_t gate_stride,
                          const uint16_t* pre_w, void* h_out, int64_t h_out_stride, uint16_t* hn,
                          int64_t hn_stride, void* stream) {
  if (!desc) return mfail(GDN_ERR_INVALID, "gdn_block_norm: NULL descriptor");
  const gdn_block_norm_desc& d = *desc;
  if (d.hidden < 8 || d.hidden > 16384 || d.hidden % 8 != 0)
    return mfail(GDN_ERR_UNSUPPORTED, "gdn_block_norm: hidden = %d not a multiple of 8 in "
                 "[8, 16384]", d.hidden);
  if (d.gate < GDN_GATE_NONE || d.gate > GDN_GATE_ELEMENT)
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: gate = %d", d.gate);
  if (!(d.post_eps >= 0.0f) || !(d.pre_eps >= 0.0f))
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: post_eps and pre_eps must be >= 0");
  if (n < 0) return mfail(GDN_ERR_INVALID, "gdn_block_norm: n = %d < 0", n);
  if (n == 0) return GDN_OK;
  if (!h || !x || !h_out) return mfail(GDN_ERR_INVALID, "gdn_block_norm: NULL tensor pointer");
  if (!pre_w != !hn)
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: pre_w and hn go together (one is NULL)");
  if ((d.gate != GDN_GATE_NONE) != (gate != nullptr))
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: gate tensor and gate = %d do not agree", d.gate);
  const struct {
    const char* name;
    const void* p;
    int64_t stride;
  } rows[] = {{"h", h, h_stride}, {"x", x, x_stride}, {"h_out", h_out, h_out_stride},
              {"hn", hn, hn_stride}};
  for (const auto& r : rows)
    if (r.p && (!aligned(r.p, 16) || r.stride < d.hidden || r.stride % 8 != 0))
      return mfail(GDN_ERR_INVALID, "gdn_block_norm: %s needs 16-byte alignment and a row stride "
                   ">= %d that is a multiple of 8 (got %lld)", r.name, d.hidden,
                   (long long)r.stride);
  if (!aligned(post_w, 16) || !aligned(pre_w, 16))
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: the norm weights need 16-byte alignment");
  if (d.gate == GDN_GATE_ELEMENT &&
      (!aligned(gate, 16) || gate_stride % 8 != 0 ||
       (gate_stride != 0 && gate_stride < d.hidden)))
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: an element gate needs 16-byte alignment and a "
                 "row stride of 0 or a multiple of 8 >= %d (got %lld)", d.hidden,
                 (long long)gate_stride);
  if (d.gate == GDN_GATE_ROW && (gate_stride < 0 || !aligned(gate, 2)))
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: a row gate needs a stride >= 0 (got %lld)",
                 (long long)gate_stride);
  if ((h == h_out && h_stride != h_out_stride) || (x == hn && x_stride != hn_stride))
    return mfail(GDN_ERR_INVALID, "gdn_block_norm: a tensor updated in place keeps its stride");
  gdn::BlockNormArgs a{};
  a.d = d;
  a.h_stride = h_stride;
  a.h_out_stride = h_out_stride;
  a.x_stride = x_stride;
  a.post_w = post_w;
  a.gate_stride = gate_stride;
  a.pre_w = pre_w;
  a.hn_stride = hn_stride;
  a.stream = static_cast<hipStream_t>(stream);
  const int64_t hb = d.h_f32 ? 4 : 2;
  for (int64_t i = 0; i < n; i += kRowsOfLaunch) {
    a.n = (int)std::min<int64_t>(n - i, kRowsOfLaunch);
    a.h = static_cast<const char*>(h) + i * h_stride * hb;
    a.h_out = static_cast<char*>(h_out) + i * h_out_stride * hb;
    a.x = x + i * x_stride;
    a.gate = gate ? gate + i * gate_stride : nullptr;
    a.hn = hn ? hn + i * hn_stride : nullptr;
    const hipError_t e = gdn::launch_block_norm(a);
    if (e != hipSuccess) return hip_fail(e, "gdn_block_norm launch");
  }
  return GDN_OK;
}

}  // extern "C"
