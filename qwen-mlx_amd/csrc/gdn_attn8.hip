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
  float slope;    // of the lane's column, * log2(e), or 0
};

// softcap * tanh(y): 1 - 2 / (1 + e^2y), off by some 2^-23 of the cap
__device__ __forceinline__ float capped(float y, float cap) {
  const float e = __builtin_amdgcn_exp2f(y * 2.8853900817779268f);  // e^2y; inf: 1
  return cap * fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
}

// Rows of the step: for group g of the `tpg`-token groups of all rows in order, its row and
// the row's first group.
struct Row {
  int r, slot, pos, fresh, first;
};

// The row that item g lies in, where row r has items(r) of them; first: its first item. By
// the wave. r = -1: none.
template <typename F>
__device__ __forceinline__ Row find_row(const Kv8Plan& p, int g, F items) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  Row w{-1, -1, 0, 0, 0};
  for (int b = 0; b < p.n; b += 64) {
    const int r = b + lane;
    const bool in = r < p.n;
    const int pos = in ? p.row_pos[r] : 0, fresh = in ? p.row_new[r] : 0;
    const int mine = in ? items(r, pos, fresh) : 0;
    int s = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int u = __shfl_up(s, off, 64);
      s += lane >= off ? u : 0;
    }
    const int total = __builtin_amdgcn_readlane(s, 63);
    if (g < base + total) {
      const int l = __popcll(__ballot(base + s <= g));
      w.r = b + l;
      w.pos = __builtin_amdgcn_readlane(pos, l);
      w.fresh = __builtin_amdgcn_readlane(fresh, l);
      w.first = base + __builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(mine, l);
      w.slot = p.row_slot[w.r];
      return w;
    }
    base += total;
  }
  return w;
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

// sigmoid of a gate, times o
__device__ __forceinline__ float gated(float o, float g) { return o * sigmoid_f32(g); }

}  // namespace

// One wave per (group of up to 16 / G tokens of a row, kv head): the 16 columns of the tiles
// are (token, query head) pairs, column c = token c / G, head c % G. Each wave goes through all
// pages that its tokens see.
template <int D>
__global__ __launch_bounds__(64) void attn8_rows_kernel(Kv8AttnArgs a) {
  constexpr int NK = D / 64, DB = D / 16;
  const Kv8Plan& p = a.p;
  const int lane = threadIdx.x, g4 = lane >> 4, c = lane & 15;
  const int G = p.Hq / p.Hkv, tpg = 16 / G, j = blockIdx.y;
  const int g = blockIdx.x;
  const Row w = find_row(p, g, [&](int, int, int fresh) { return (fresh + tpg - 1) / tpg; });
  if (w.r < 0) return;
  const int k0 = (g - w.first) * tpg;             // first token of the row
  const int nt = min(tpg, w.fresh - k0);
  const int pos0 = w.pos + k0, total = w.pos + w.fresh;
  const int ctok = c / G, h = j * G + c % G;
  const bool valid = ctok < nt;
  const int64_t t = p.cu[w.r] + k0 + (valid ? ctok : 0);
  const int cpos = valid ? pos0 + ctok : -1;
  const int pf = a.prefix ? min(max(a.prefix[w.r], 0), total) : 0;
  const int lo = a.window > 0 ? cpos - a.window : -1;  // keys above it
  const Span span = span_of(pos0, pos0 + nt - 1, a.window, pf, total);
  Score sc;
  sc.mul = a.softcap > 0.f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
  sc.cap = a.softcap * 1.4426950408889634f;
  sc.slope = a.slopes ? a.slopes[valid ? h : 0] * 1.4426950408889634f : 0.f;

  u32x4 q[NK][2];
#pragma unroll
  for (int i = 0; i < NK; ++i)
#pragma unroll
    for (int b = 0; b < 2; ++b)
      q[i][b] = valid ? *reinterpret_cast<const u32x4*>(a.q + t * a.qs + h * a.qhs + 64 * i + 16 * g4 + 8 * b)
                      : (u32x4){0u, 0u, 0u, 0u};

  float m = -INFINITY, l = 0.f;
  f32x4 O[DB];
  int unit = 0;
#pragma unroll
  for (int d = 0; d < DB; ++d) O[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int32_t* const row = p.table + (size_t)w.slot * p.max_pages;
  for (int v = 0; v < span.count(); ++v) {
    const int blk = span.page(v), key0 = blk * kPage;
    const size_t hk = ((size_t)row[blk] * 2) * p.Hkv + j, hv = hk + p.Hkv;
    const u32x4* const kp = reinterpret_cast<const u32x4*>(a.pages + hk * (kPage * D)) + lane;
    const u32x4* const vp = reinterpret_cast<const u32x4*>(a.pages + hv * (kPage * D)) + lane;
    const int ek = (int)(int8_t)a.exps[hk], wv = a.exps[hv], ev = (int)(int8_t)wv;
    f32x4 S[4];
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) {
      S[kg] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const u32x4 kr = kp[(kg * NK + i) * 64];
        S[kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            to_bf16(kr[0], kr[1]), __builtin_bit_cast(bf16x8, q[i][0]), S[kg], 0, 0, 0);
        S[kg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            to_bf16(kr[2], kr[3]), __builtin_bit_cast(bf16x8, q[i][1]), S[kg], 0, 0, 0);
      }
    }
    // scores of keys key0 + 16 kg + 4 g4 + r
    float x[16], bm = -INFINITY;
    const float mul = sc.mul * pow2(ek);
#pragma unroll
    for (int kg = 0; kg < 4; ++kg)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = key0 + 16 * kg + 4 * g4 + r;
        float y = S[kg][r] * mul;
        if (sc.cap > 0.f) y = capped(y, sc.cap);
        y = fmaf(-sc.slope, (float)(cpos - key), y);
        const bool see = (key <= cpos && key > lo) || (key < pf && valid);
        x[4 * kg + r] = see ? y : -INFINITY;
        bm = fmaxf(bm, x[4 * kg + r]);
      }
    const float mn = fmaxf(m, max_xor16_32(bm));
    float corr = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;  // m = -inf: 0
    m = mn;
    l *= corr;
    corr *= v ? __builtin_amdgcn_ldexpf(1.0f, unit - ev) : 1.0f;
    unit = ev;
#pragma unroll
    for (int d = 0; d < DB; ++d) O[d] *= corr;
    const float mref = m == -INFINITY ? 0.f : m;
    u32x4 P[2];
    uint32_t seen = 0;
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) {
      float e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] = __builtin_amdgcn_exp2f(x[4 * kg + r] - mref);
        seen |= (x[4 * kg + r] != -INFINITY ? 1u : 0u) << (4 * kg + r);
      }
      l += (e[0] + e[1]) + (e[2] + e[3]);
      P[kg >> 1][(kg & 1) * 2] = pk_f16(e[0], e[1]);
      P[kg >> 1][(kg & 1) * 2 + 1] = pk_f16(e[2], e[3]);
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      u32x4 vr = vp[d * 64];
      if (key0 + kPage > total) {  // keys past the row's end may hold anything
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) {
          const int n = total - (key0 + 16 * kg + 4 * g4);
          vr[kg] &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        }
      }
      f16x8 v0 = to_f16(vr[0], vr[1]), v1 = to_f16(vr[2], vr[3]);
      if (wv & kNanFlag) {
        // NaN values reach the columns that see their keys, and no others: they leave the
        // product, and a second one counts them
        f16x8 n0, n1, s0, s1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          n0[i] = v0[i] == v0[i] ? (_Float16)0.f : (_Float16)1.f;
          n1[i] = v1[i] == v1[i] ? (_Float16)0.f : (_Float16)1.f;
          v0[i] = v0[i] == v0[i] ? v0[i] : (_Float16)0.f;
          v1[i] = v1[i] == v1[i] ? v1[i] : (_Float16)0.f;
          s0[i] = (seen >> i) & 1u ? (_Float16)1.f : (_Float16)0.f;
          s1[i] = (seen >> (8 + i)) & 1u ? (_Float16)1.f : (_Float16)0.f;
        }
        f32x4 cnt = {0.f, 0.f, 0.f, 0.f};
        cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(n0, s0, cnt, 0, 0, 0);
        cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(n1, s1, cnt, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) O[d][r] = cnt[r] > 0.f ? __builtin_nanf("") : O[d][r];
      }
      O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, __builtin_bit_cast(f16x8, P[0]), O[d], 0, 0, 0);
      O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, __builtin_bit_cast(f16x8, P[1]), O[d], 0, 0, 0);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (!valid) return;
  const float inv = __builtin_amdgcn_ldexpf(1.0f / l, unit);
#pragma unroll
  for (int d = 0; d < DB; ++d) {
    const int dim = 16 * d + 4 * g4;
    float o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = O[d][r] * inv;
    if (a.gate) {
      const u32x2 gv = *reinterpret_cast<const u32x2*>(a.gate + t * a.gs + h * a.ghs + dim);
      o[0] = gated(o[0], bf_lo(gv.x));
      o[1] = gated(o[1], bf_hi(gv.x));
      o[2] = gated(o[2], bf_lo(gv.y));
      o[3] = gated(o[3], bf_hi(gv.y));
    }
    *reinterpret_cast<u32x2*>(a.out + t * a.os + h * a.ohs + dim) =
        (u32x2){f2bf2(o[0], o[1]), f2bf2(o[2], o[3])};
  }
}

// Tokens of refused rows: zeros. grid T, block 256.
__global__ __launch_bounds__(256) void attn8_zero_kernel(Kv8AttnArgs a) {
  const Kv8Plan& p = a.p;
  const int64_t t = blockIdx.x;
  if (t >= p.cu[p.n] || p.pos[t] >= 0) return;
  const int per = p.D / 4;
  for (int i = threadIdx.x; i < p.Hq * per; i += 256)
    *reinterpret_cast<u32x2*>(a.out + t * a.os + (i / per) * a.ohs + (i % per) * 4) = (u32x2){0u, 0u};
}

size_t kv8_attn_workspace_bytes(const gdn_kv8_desc&) { return 0; }

hipError_t launch_kv8_attn(const Kv8AttnArgs& a) {
  const Kv8Plan& p = a.p;
  const int tpg = 16 / (p.Hq / p.Hkv);
  hipLaunchKernelGGL(attn8_zero_kernel, dim3(p.T), dim3(256), 0, a.stream, a);
  const dim3 grid(min(p.T, p.T / tpg + min(p.n, p.T)), p.Hkv);
  if (p.D == 256)
    hipLaunchKernelGGL(attn8_rows_kernel<256>, grid, dim3(64), 0, a.stream, a);
  else if (p.D == 128)
    hipLaunchKernelGGL(attn8_rows_kernel<128>, grid, dim3(64), 0, a.stream, a);
  else
    hipLaunchKernelGGL(attn8_rows_kernel<64>, grid, dim3(64), 0, a.stream, a);
  return hipGetLastError();
}

}  // namespace gdn
