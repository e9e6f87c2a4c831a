// gdn_attn8.hip -- attention over the 8-bit paged cache (layout: gdn_kv8.hip).
// For the query of head h at position i and the key at position j
//   s = softcap(scale * q . k) - slope_h (i - j),  out = sum_j softmax(s)_j v_j
// over the visible j, with one pass over the keys and the running maximum and sum of
// the softmax.
//
// Scores and P V run on MFMA. e4m3 numbers convert exactly into bf16 (for q . k with q as
// it is) and into f16 (for P V: P in [0, 1] as f16 keeps 11 bits, three more than
// bf16), both without their page's exponent: the keys' exponent multiplies the scores, the
// values' is the unit of the running outputs, which are rescaled where it changes.
#include "gdn_common.h"

namespace gdn {

namespace {

constexpr int kPage = 64;
constexpr int kNanFlag = 1 << 16;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// 8 e4m3 bytes to 8 bf16 / 8 f16 (both exact)
__device__ __forceinline__ bf16x8 to_bf16(uint32_t a, uint32_t b) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
  return __builtin_bit_cast(bf16x8, r);
}
__device__ __forceinline__ f16x8 to_f16(uint32_t a, uint32_t b) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
  return __builtin_bit_cast(f16x8, r);
}
__device__ __forceinline__ uint32_t pk_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}

// Maximum over the four lanes of a column (lane ^ 16, lane ^ 32, both).
__device__ __forceinline__ float max_xor16_32(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// What a call adds to the scores, in the log2 domain: x = f(s * 2^ek).
struct Score {
  float mul;      // scale * log2(e), or scale / softcap
  float cap;      // softcap * log2(e), or 0
  float slope;    // of the lane's column, * log2(e)
  bool sloped;
  int window;     // or more than any position
};

// softcap * tanh(y): 1 - 2 / (1 + e^2y), off by some 2^-23 of the cap
__device__ __forceinline__ float capped(float y, float cap) {
  const float e = __builtin_amdgcn_exp2f(y * 2.8853900817779268f);  // e^2y; inf: 1
  return cap * fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int s) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int u = __shfl_up(s, off, 64);
    s += lane >= off ? u : 0;
  }
  return s;
}

struct Found {
  int r, first;  // row and its first item; r = -1: none
  Kv8Row row;
};

// The row that item g lies in, where a row has items(r, row) of them, by the wave. `before`
// and b0: items of the rows before row b0 (a multiple of 64).
template <typename F>
__device__ __forceinline__ Found find_row(const Kv8Plan& p, int g, int b0, int before, F items) {
  const int lane = threadIdx.x & 63;
  for (int b = b0; b < p.n; b += 64) {
    const int r = b + lane;
    const Kv8Row row = r < p.n ? p.rows[r] : Kv8Row{-1, 0, 0, 0};
    const int mine = row.fresh > 0 ? items(r, row) : 0;
    const int s = wave_scan(mine);
    const int total = __builtin_amdgcn_readlane(s, 63);
    if (g < before + total) {
      const int l = __popcll(__ballot(before + s <= g));
      Found f;
      f.r = b + l;
      f.first = before + __builtin_amdgcn_readlane(s - mine, l);
      f.row = Kv8Row{__builtin_amdgcn_readlane(row.slot, l), __builtin_amdgcn_readlane(row.pos, l),
                     __builtin_amdgcn_readlane(row.fresh, l), __builtin_amdgcn_readlane(row.cu, l)};
      return f;
    }
    before += total;
  }
  return Found{-1, 0, {-1, 0, 0, 0}};
}

// Visible keys of a group of tokens, as pages: [0, pre) then [lo, end).
struct Span {
  int pre, lo, end;
  __device__ __forceinline__ int count() const { return pre + end - lo; }
  __device__ __forceinline__ int page(int v) const { return v < pre ? v : v - pre + lo; }
};
// p0, p1: first and last position; total: the row's length with the step; pf: its prefix
__device__ __forceinline__ Span span_of(int p0, int p1, int window, int pf, int total) {
  Span s;
  const int keys = min(max(p1 + 1, pf), total);
  s.end = (keys + kPage - 1) / kPage;
  s.lo = window > 0 ? max(p0 - window + 1, 0) / kPage : 0;
  s.pre = min((pf + kPage - 1) / kPage, s.lo);
  return s;
}

// Four outputs of a head from dim on: times sigmoid(gate) where there is one, rounded once.
__device__ __forceinline__ void store4(const Kv8AttnArgs& a, int64_t t, int h, int dim, float* o) {
  if (a.gate) {
    const u32x2 g = *reinterpret_cast<const u32x2*>(a.gate + t * a.gs + h * a.ghs + dim);
    o[0] *= sigmoid_f32(bf_lo(g.x));
    o[1] *= sigmoid_f32(bf_hi(g.x));
    o[2] *= sigmoid_f32(bf_lo(g.y));
    o[3] *= sigmoid_f32(bf_hi(g.y));
  }
  *reinterpret_cast<u32x2*>(a.out + t * a.os + h * a.ohs + dim) =
      (u32x2){f2bf2(o[0], o[1]), f2bf2(o[2], o[3])};
}

// V bytes of a lane: the A operands of dims 2 i and 2 i + 1 (of 16), 32 keys.
__device__ __forceinline__ void v_operands(u32x4 v, u32x2& a, u32x2& b) {
  const auto x = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  a = (u32x2){x[0], y[0]};
  b = (u32x2){x[1], y[1]};
}

// Bytes of keys from `left` keys on taken out: n = keys that remain from the word's first.
__device__ __forceinline__ uint32_t first_keys(uint32_t w, int n) {
  return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u);
}

// What a group of tokens of a row reads: 16 columns (token, query head of kv head j).
struct Group {
  int h, cpos, lo, pf, total, pos0, nt;
  int64_t t;
  bool valid;
  Span span;
};
__device__ __forceinline__ Group group_of(const Kv8AttnArgs& a, const Kv8Row& row, int r, int g, int j,
                                          int G, int tpg, int c) {
  Group x;
  const int k0 = g * tpg, ctok = c / G;
  x.nt = min(tpg, row.fresh - k0);
  x.pos0 = row.pos + k0;
  x.total = row.pos + row.fresh;
  x.valid = ctok < x.nt;
  x.h = j * G + c % G;
  x.t = (int64_t)row.cu + k0 + (x.valid ? ctok : 0);
  x.cpos = x.valid ? x.pos0 + ctok : -1;
  x.pf = a.prefix ? min(max(a.prefix[r], 0), x.total) : 0;
  x.lo = a.window > 0 ? x.cpos - a.window : -1;  // keys above it
  x.span = span_of(x.pos0, x.pos0 + x.nt - 1, a.window, x.pf, x.total);
  return x;
}

// The running softmax of 16 columns: lane (g4, c) holds keys 16 kg + 4 g4 + r of a page for
// column c, and dims 16 d + 4 g4 + r of its outputs in units of 2^unit.
template <int D>
struct Online {
  float m, l;
  int unit;
  f32x4 O[D / 16];

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
    unit = 0;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) O[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }

  // Scores S of the page at key0 to weights P; ek, ev: the exponents of its keys and values
  __device__ __forceinline__ void weights(const f32x4* S, const Score& sc, const Group& x, int key0,
                                          int ek, int ev, u32x4* P, uint32_t& seen) {
    const int g4 = (threadIdx.x & 63) >> 4;
    float s[16], bm = -INFINITY;
    const float mul = sc.mul * pow2(ek);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = S[i >> 2][i & 3] * mul;
    if (sc.cap > 0.f) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = capped(s[i], sc.cap);
    }
    if (sc.sloped) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = fmaf(-sc.slope, (float)(x.cpos - (key0 + 16 * (i >> 2) + 4 * g4 + (i & 3))), s[i]);
    }
    seen = 0xffffu;
    // wave-uniform: every token of the group sees every key of the page
    const bool all = (key0 + kPage - 1 <= x.pos0 && key0 > x.pos0 + x.nt - 1 - sc.window) ||
                     key0 + kPage <= x.pf;
    if (!all) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = key0 + 16 * (i >> 2) + 4 * g4 + (i & 3);
        const bool see = (key <= x.cpos && key > x.lo) || (key < x.pf && x.valid);
        s[i] = see ? s[i] : -INFINITY;
        seen &= ~((see ? 0u : 1u) << i);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) bm = fmaxf(bm, s[i]);
    bm = max_xor16_32(bm);
    if (__any(bm > m) || ev != unit) {
      const float mn = fmaxf(m, bm);
      float corr = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;  // m = -inf: 0
      m = mn;
      l *= corr;
      corr = __builtin_amdgcn_ldexpf(corr, unit - ev);
      unit = ev;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) O[d] *= corr;
    }
    const float mref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) {
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(s[4 * kg + r] - mref);
      l += (e[0] + e[1]) + (e[2] + e[3]);
      P[kg >> 1][(kg & 1) * 2] = pk_f16(e[0], e[1]);
      P[kg >> 1][(kg & 1) * 2 + 1] = pk_f16(e[2], e[3]);
    }
  }

  // O[d] += the operand's 16 dims x 32 keys (half p of the page) . P
  __device__ __forceinline__ void values(int d, u32x2 v, u32x4 P, const Group& x, int key0, int p,
                                         bool has_nan, uint32_t seen) {
    const int g4 = (threadIdx.x & 63) >> 4;
    if (key0 + kPage > x.total) {  // keys past the row's end may hold anything
      const int n = x.total - (key0 + 32 * p + 4 * g4);
      v.x = first_keys(v.x, n);
      v.y = first_keys(v.y, n - 16);
    }
    f16x8 f = to_f16(v.x, v.y);
    if (has_nan) {
      // NaN values reach the columns that see their keys, and no others: they leave the
      // product, and another one counts them
      f16x8 bad, eye;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bad[i] = f[i] == f[i] ? (_Float16)0.f : (_Float16)1.f;
        f[i] = f[i] == f[i] ? f[i] : (_Float16)0.f;
        eye[i] = (seen >> (8 * p + i)) & 1u ? (_Float16)1.f : (_Float16)0.f;
      }
      const f32x4 cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, eye, (f32x4){0.f, 0.f, 0.f, 0.f},
                                                               0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) O[d][r] = cnt[r] > 0.f ? __builtin_nanf("") : O[d][r];
    }
    O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, __builtin_bit_cast(f16x8, P), O[d], 0, 0, 0);
  }

  __device__ __forceinline__ float sum() const {
    const float s = l + __shfl_xor(l, 16, 64);
    return s + __shfl_xor(s, 32, 64);
  }
};

__device__ __forceinline__ Score score_of(const Kv8AttnArgs& a, const Group& x) {
  Score sc;
  sc.mul = a.softcap > 0.f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
  sc.cap = a.softcap * 1.4426950408889634f;
  sc.sloped = a.slopes != nullptr;
  sc.slope = a.slopes ? a.slopes[x.valid ? x.h : 0] * 1.4426950408889634f : 0.f;
  sc.window = a.window > 0 ? a.window : INT32_MAX / 2;
  return sc;
}

// Items of a row of few tokens: (group, kv head, chunk) in this order.
struct Chunks {
  int groups, cp, nch;
};
__device__ __forceinline__ Chunks chunks_of(const Kv8AttnArgs& a, const Kv8Row& row, int r, int tpg) {
  Chunks c{0, 1, 0};
  if (row.fresh <= 0 || row.fresh >= kKv8TileTokens) return c;
  c.groups = (row.fresh + tpg - 1) / tpg;
  c.cp = kv8_chunk_pages(c.groups);
  const int total = row.pos + row.fresh;
  const int pf = a.prefix ? min(max(a.prefix[r], 0), total) : 0;
  // the first and the last group's pages; one between them may see a page more where the
  // window's two ends fall into pages
  int most = 0;
  for (int g = 0; g < c.groups; g += max(c.groups - 1, 1)) {
    const int p0 = row.pos + g * tpg;
    most = max(most, span_of(p0, min(p0 + tpg, total) - 1, a.window, pf, total).count());
  }
  most = min(most + (c.groups > 1 && a.window > 0 ? 1 : 0), (total + kPage - 1) / kPage);
  c.nch = (most + c.cp - 1) / c.cp;
  return c;
}

}  // namespace

// One wave per work-group; worker w of P takes the chunks [w k, (w + 1) k) of all rows' items,
// k = ceil(items / P), each chunk its own partial: a token's result depends on its own row
// alone. The next page's keys are loaded as soon as this page's scores are formed, its
// values after this page's products, across chunks of a segment.
template <int D>
__global__ __launch_bounds__(64, D == 256 ? 1 : 2) void attn8_chunk_kernel(Kv8AttnArgs a, float* __restrict__ part) {
  constexpr int NK = D / 64, DB = D / 16;
  __shared__ u32x4 qlds[2 * NK][64];
  __shared__ int before[kKv8Rows / 64];
  const Kv8Plan& p = a.p;
  const int lane = threadIdx.x, g4 = lane >> 4, c = lane & 15;
  const int G = p.Hq / p.Hkv, tpg = 16 / G;
  auto items = [&](int r, const Kv8Row& row) {
    const Chunks k = chunks_of(a, row, r, tpg);
    return k.groups * k.nch * p.Hkv;
  };
  int all = 0;
  for (int b = 0; b < p.n; b += 64) {
    const int r = b + lane;
    int mine = 0;
    if (r < p.n) mine = items(r, p.rows[r]);
    if (lane == 0) before[b >> 6] = all;
    all += __builtin_amdgcn_readlane(wave_scan(mine), 63);
  }
  const int k = (all + gridDim.x - 1) / gridDim.x;
  int g = blockIdx.x * k;
  const int gend = min(all, g + k);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  while (g < gend) {
    int b = 0;
    while (b + 64 < p.n && before[(b >> 6) + 1] <= g) b += 64;
    const Found f = find_row(p, g, b, before[b >> 6], items);
    const Chunks ch = chunks_of(a, f.row, f.r, tpg);
    const int local = g - f.first, seg = local / ch.nch, c0 = local - seg * ch.nch;
    const int grp = seg / p.Hkv, j = seg - grp * p.Hkv;
    const int nc = min(gend - g, ch.nch - c0);  // chunks of this segment
    g += nc;
    const Group x = group_of(a, f.row, f.r, grp, j, G, tpg, c);
    const Score sc = score_of(a, x);
    const int count = x.span.count();
    const int v1 = min((c0 + nc) * ch.cp, count);
    float* const out = part + ((size_t)p.parts[f.r] * p.Hkv + (size_t)seg * ch.nch) * (16 * (D + 4));
    {
      const uint16_t* const q = a.q + x.t * a.qs + x.h * a.qhs + 16 * g4;
#pragma unroll
      for (int i = 0; i < 2 * NK; ++i)
        qlds[i][lane] = x.valid ? *reinterpret_cast<const u32x4*>(q + 64 * (i >> 1) + 8 * (i & 1))
                                : (u32x4){0u, 0u, 0u, 0u};
    }
    const int32_t* const trow = p.table + (size_t)f.row.slot * p.max_pages;
    // ids and exponents of 64 pages, one a lane
    int vbase = 0, pid = 0, eks = 0, evs = 0;
    auto ids = [&](int v) {
      vbase = v;
      pid = v + lane < v1 ? trow[x.span.page(v + lane)] : 0;
      const int32_t* const e = a.exps + (size_t)pid * 2 * p.Hkv + j;
      eks = e[0];
      evs = e[p.Hkv];
    };
    const uint8_t* const base = a.pages + (size_t)j * (kPage * D) + lane * 16;
    const size_t page_bytes = (size_t)2 * p.Hkv * kPage * D, v_shift = (size_t)p.Hkv * kPage * D;
    u32x4 kf[4 * NK], vf[DB];
    auto page_of = [&](int v) {
      return base + (size_t)(uint32_t)__builtin_amdgcn_readlane(pid, v - vbase) * page_bytes;
    };
    auto load_k = [&](const uint8_t* s) {
#pragma unroll
      for (int i = 0; i < 4 * NK; ++i)
        kf[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(s) + i * 64);
    };
    auto load_v = [&](const uint8_t* s) {
#pragma unroll
      for (int i = 0; i < DB; ++i)
        vf[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(s + v_shift) + i * 64);
    };
    Online<D> on;
    on.clear();
    auto flush = [&](int chunk) {
      const float l = on.sum();
      if (ch.nch == 1) {
        if (!x.valid) return;
        const float inv = __builtin_amdgcn_ldexpf(1.0f / l, on.unit);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          float o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = on.O[d][r] * inv;
          store4(a, x.t, x.h, 16 * d + 4 * g4, o);
        }
      } else if (x.valid) {
        float* const pr = out + ((size_t)chunk * 16 + c) * (D + 4);
        if (g4 == 0) {
          pr[0] = on.m;
          pr[1] = l;
        }
        const float one = __builtin_amdgcn_ldexpf(1.0f, on.unit);
#pragma unroll
        for (int d = 0; d < DB; ++d)
          *reinterpret_cast<f32x4*>(pr + 4 + 16 * d + 4 * g4) = on.O[d] * one;
      }
      on.clear();
    };
    int v = c0 * ch.cp;
    if (v < v1) {
      ids(v);
      const uint8_t* cur = page_of(v);
      load_k(cur);
      load_v(cur);
    }
    for (int chunk = c0; chunk < c0 + nc; ++chunk) {
      const int vend = min((chunk + 1) * ch.cp, v1);
      for (; v < vend; ++v) {
        const int key0 = x.span.page(v) * kPage;
        const int ek = (int)(int8_t)__builtin_amdgcn_readlane(eks, v - vbase);
        const int wv = __builtin_amdgcn_readlane(evs, v - vbase), ev = (int)(int8_t)wv;
        if (v + 1 < v1 && v + 1 - vbase >= 64) ids(v + 1);
        const uint8_t* const nxt = page_of(min(v + 1, v1 - 1));
        f32x4 S[4];
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) S[kg] = (f32x4){0.f, 0.f, 0.f, 0.f};
        asm volatile("" ::: "memory");  // q is re-read from LDS for every page
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const bf16x8 q0 = __builtin_bit_cast(bf16x8, qlds[2 * i][lane]);
          const bf16x8 q1 = __builtin_bit_cast(bf16x8, qlds[2 * i + 1][lane]);
#pragma unroll
          for (int kg = 0; kg < 4; ++kg) {
            const u32x4 kr = kf[kg * NK + i];
            S[kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(kr[0], kr[1]), q0, S[kg], 0, 0, 0);
            S[kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(kr[2], kr[3]), q1, S[kg], 0, 0, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (v + 1 < v1) load_k(nxt);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 P[2];
        uint32_t seen;
        on.weights(S, sc, x, key0, ek, ev, P, seen);
        const bool has_nan = (wv & kNanFlag) != 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < DB / 2; ++i) {
            u32x2 va, vb;
            v_operands(vf[h * (DB / 2) + i], va, vb);
            on.values(2 * i, va, P[h], x, key0, h, has_nan, seen);
            on.values(2 * i + 1, vb, P[h], x, key0, h, has_nan, seen);
          }
        __builtin_amdgcn_sched_barrier(0);
        if (v + 1 < v1) load_v(nxt);
        __builtin_amdgcn_sched_barrier(0);
      }
      flush(chunk);
    }
  }
}

// grid (T, Hq), block 256: the chunks of a token's head, each wave every fourth one, then the
// waves' sums in order. Also the zeros of refused rows' tokens. Tokens of tiles and of single
// chunks are written already.
template <int D>
__global__ __launch_bounds__(256) void attn8_combine_kernel(Kv8AttnArgs a,
                                                            const float* __restrict__ part) {
  constexpr int DPL = D / 64;
  typedef float fvec __attribute__((ext_vector_type(DPL)));
  __shared__ float sum[4][D];
  const Kv8Plan& p = a.p;
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = p.tok_row[t];
  if (r == -2) return;
  if (r < 0) {
    if (tid < D / 4)
      *reinterpret_cast<u32x2*>(a.out + (int64_t)t * a.os + h * a.ohs + 4 * tid) = (u32x2){0u, 0u};
    return;
  }
  const Kv8Row row = p.rows[r];
  const int G = p.Hq / p.Hkv, tpg = 16 / G;
  const Chunks ch = chunks_of(a, row, r, tpg);
  if (ch.nch < 2) return;
  const int k = t - row.cu, grp = k / tpg, j = h / G, c = (k - grp * tpg) * G + h - j * G;
  const float* const pc = part + (((size_t)p.parts[r] * p.Hkv + (size_t)(grp * p.Hkv + j) * ch.nch) *
                                      16 + c) * (D + 4);
  constexpr size_t kStride = (size_t)16 * (D + 4);
  float M = -INFINITY;
  for (int i = lane; i < ch.nch; i += 64) M = fmaxf(M, pc[i * kStride]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  if (M == -INFINITY) M = 0.f;  // NaN scores alone
  float L = 0.f;
  fvec A = (fvec)(0.f);
  for (int i0 = 0; i0 < ch.nch; i0 += 64) {
    const int n = min(64, ch.nch - i0);
    const float* const ps = pc + (size_t)i0 * kStride;
    const float w = lane < n ? exp2f(ps[lane * kStride] - M) : 0.f;
    const float l = lane < n ? ps[lane * kStride + 1] : 0.f;
    L += l != 0.f ? w * l : 0.f;
    for (int i = wave; i < n; i += 4) {
      const float wi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), i));
      const float li = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l), i));
      // a chunk without a visible key may hold anything
      const fvec v = *reinterpret_cast<const fvec*>(ps + i * kStride + 4 + DPL * lane);
      if (li != 0.f) A += v * wi;
    }
  }
  L = wave_sum(L);
#pragma unroll
  for (int i = 0; i < DPL; ++i) sum[wave][DPL * lane + i] = A[i];
  __syncthreads();
  if (tid < D / 4) {
    const float inv = 1.0f / L;
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 4 * tid + i;
      o[i] = ((sum[0][d] + sum[1][d]) + (sum[2][d] + sum[3][d])) * inv;
    }
    store4(a, t, h, 4 * tid, o);
  }
}

// One wave per (group of up to 16 / G tokens of a row of many, kv head) through all pages that its
// tokens see.
template <int D>
__global__ __launch_bounds__(64) void attn8_rows_kernel(Kv8AttnArgs a) {
  constexpr int NK = D / 64, DB = D / 16;
  const Kv8Plan& p = a.p;
  const int lane = threadIdx.x, g4 = lane >> 4, c = lane & 15;
  const int G = p.Hq / p.Hkv, tpg = 16 / G, j = blockIdx.y;
  const int g = blockIdx.x;
  const Found f = find_row(p, g, 0, 0, [&](int, const Kv8Row& row) {
    return row.fresh < kKv8TileTokens ? 0 : (row.fresh + tpg - 1) / tpg;
  });
  if (f.r < 0) return;
  const Group x = group_of(a, f.row, f.r, g - f.first, j, G, tpg, c);
  const Score sc = score_of(a, x);
  u32x4 q[2 * NK];
#pragma unroll
  for (int i = 0; i < 2 * NK; ++i)
    q[i] = x.valid ? *reinterpret_cast<const u32x4*>(a.q + x.t * a.qs + x.h * a.qhs + 64 * (i >> 1) +
                                                     16 * g4 + 8 * (i & 1))
                   : (u32x4){0u, 0u, 0u, 0u};
  Online<D> on;
  on.clear();
  const int32_t* const trow = p.table + (size_t)f.row.slot * p.max_pages;
  for (int v = 0; v < x.span.count(); ++v) {
    const int blk = x.span.page(v), key0 = blk * kPage;
    const size_t hk = ((size_t)trow[blk] * 2) * p.Hkv + j, hv = hk + p.Hkv;
    const u32x4* const kp = reinterpret_cast<const u32x4*>(a.pages + hk * (kPage * D)) + lane;
    const u32x4* const vp = reinterpret_cast<const u32x4*>(a.pages + hv * (kPage * D)) + lane;
    const int wv = a.exps[hv];
    f32x4 S[4];
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) {
      S[kg] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const u32x4 kr = kp[(kg * NK + i) * 64];
        S[kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            to_bf16(kr[0], kr[1]), __builtin_bit_cast(bf16x8, q[2 * i]), S[kg], 0, 0, 0);
        S[kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            to_bf16(kr[2], kr[3]), __builtin_bit_cast(bf16x8, q[2 * i + 1]), S[kg], 0, 0, 0);
      }
    }
    u32x4 P[2];
    uint32_t seen;
    on.weights(S, sc, x, key0, (int)(int8_t)a.exps[hk], (int)(int8_t)wv, P, seen);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < DB / 2; ++i) {
        u32x2 va, vb;
        v_operands(vp[(h * (DB / 2) + i) * 64], va, vb);
        on.values(2 * i, va, P[h], x, key0, h, (wv & kNanFlag) != 0, seen);
        on.values(2 * i + 1, vb, P[h], x, key0, h, (wv & kNanFlag) != 0, seen);
      }
  }
  const float l = on.sum();
  if (!x.valid) return;
  const float inv = __builtin_amdgcn_ldexpf(1.0f / l, on.unit);
#pragma unroll
  for (int d = 0; d < DB; ++d) {
    float o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = on.O[d][r] * inv;
    store4(a, x.t, x.h, 16 * d + 4 * g4, o);
  }
}

size_t kv8_attn_workspace_bytes(const gdn_kv8_desc& d) {
  // chunks of a kv head over all rows of few tokens: a row has no more than its groups and one
  // for every kv8_chunk_pages(1) of its pages, which are its own
  const int64_t few = (int64_t)d.num_slots * (kKv8TileTokens - 1);
  const int64_t chunks = (few < d.max_step_tokens ? few : d.max_step_tokens) +
                         d.num_pages / kv8_chunk_pages(1) + 1;
  return (size_t)chunks * d.num_kv_heads * 16 * (d.head_dim + 4) * sizeof(float);
}

// Waves that a step of few tokens in a row is split over: those that run side by side.
template <int D>
constexpr int kWorkers = D == 256 ? 1024 : 2048;

template <int D>
static hipError_t launch_attn8(const Kv8AttnArgs& a) {
  const Kv8Plan& p = a.p;
  const int tpg = 16 / (p.Hq / p.Hkv);
  float* const part = static_cast<float*>(a.workspace);
  hipError_t e;
  if (p.max_row >= kKv8TileTokens) {
    const dim3 grid(min(p.T, p.T / tpg + min(p.n, p.T)), p.Hkv);
    hipLaunchKernelGGL(attn8_rows_kernel<D>, grid, dim3(64), 0, a.stream, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  hipLaunchKernelGGL(attn8_chunk_kernel<D>, dim3(kWorkers<D>), dim3(64), 0, a.stream, a, part);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(attn8_combine_kernel<D>, dim3(p.T, p.Hq), dim3(256), 0, a.stream, a, part);
  return hipGetLastError();
}

hipError_t launch_kv8_attn(const Kv8AttnArgs& a) {
  return a.p.D == 256 ? launch_attn8<256>(a) : a.p.D == 128 ? launch_attn8<128>(a) : launch_attn8<64>(a);
}

}  // namespace gdn
