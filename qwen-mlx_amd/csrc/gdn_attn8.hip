// gdn_attn8.hip -- attention over the 8-bit paged cache (layout: gdn_kv8.hip).
// For the query of head h at position i and the key at position j
//   s = softcap(scale * q . k) - slope_h (i - j),  out = sum_j softmax(s)_j v_j
// over the visible j, with one pass over the keys and the running maximum and sum of
// the softmax.
//
// Scores and P V run on MFMA. For q . k the keys go in as they are held, against q in two
// e4m3 parts under a power of two of its head: a bf16 number's 8 significant bits are the 4 of
// its rounding and the 4 that are left, times 16 (numbers below 2^-14 of the head's
// largest lose bits, 2^-22 of it at most). For P V the values convert exactly into f16, and P,
// in [0, 2^8] as the running maximum follows by steps of 2^8, is rounded to it: 11 bits, three
// more than bf16, and small weights by at most 2^-29 of the maximum's. The softmax's sum is of the
// rounded P, so that values that are all the same come out as they are. The pages' exponents stay
// outside: the keys' multiplies the scores; the outputs run in units of 2^(unit - 6), and P carries
// 2^(6 + the values' exponent - unit), 2^4 to 2^7: only beyond that are the outputs rescaled. With
// more f16 has no room; from 2^0 on, a million keys of weights just too small for it were lost
// beside one that weighs as much as 2^25 of them, 3% of the sum.
#include <cfloat>

#include "gdn_common.h"

namespace gdn {

namespace {

constexpr int kPage = 64;
constexpr int kBlock = 32;  // keys of a step of the running softmax: half a page
constexpr int kNanFlag = 1 << 16;
constexpr int kSplitPages = 8;  // of a tile's split at least
constexpr float kStep = 8.f;  // log2 steps of the running maximum
constexpr int kUnit = 6;      // the outputs' unit is 2^(unit - kUnit)
// Whether values of exponent ev go on in a unit: P's factor 2^(kUnit + ev - unit) is in [2^4, 2^7].
// A new unit is ev itself.
__device__ __forceinline__ bool unit_holds(int ev, int unit) {
  return ev - unit >= 4 - kUnit && ev - unit <= 7 - kUnit;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

typedef int i32x8 __attribute__((ext_vector_type(8)));

// 8 e4m3 bytes to 8 f16 (exact)
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
// s + the two f16 numbers of a word, small ones among them, in one instruction
__device__ __forceinline__ float add_f16(uint32_t two, float s) {
  const f16x2 ones = {(_Float16)1.f, (_Float16)1.f};
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, two), ones, s, false);
}

// Scores of 16 keys for 16 columns: K as held (a lane's NK 16-byte pieces of its key), q in
// two parts (NK pieces of each in turn).
template <int NK>
__device__ __forceinline__ f32x4 scores16(const u32x4* k, const u32x4* q) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if constexpr (NK >= 2) {
    constexpr int kOne = 0x7f7f7f7f, kLow = 0x7b7b7b7b;  // 2^0 and 2^-4
    auto both = [](u32x4 a, u32x4 b) {
      return (i32x8){(int)a[0], (int)a[1], (int)a[2], (int)a[3],
                     (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    };
#pragma unroll
    for (int i = 0; i < NK; i += 2) {
      const i32x8 kk = both(k[i], k[i + 1]);
      s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, both(q[2 * i], q[2 * i + 2]), s, 0, 0,
                                                           0, kOne, 0, kOne);
      s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, both(q[2 * i + 1], q[2 * i + 3]), s, 0,
                                                           0, 0, kOne, 0, kLow);
    }
  } else {
    f32x4 lo = {0.f, 0.f, 0.f, 0.f};
    auto word = [](uint32_t a, uint32_t b) { return (long)(((uint64_t)b << 32) | a); };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long kk = word(k[0][2 * h], k[0][2 * h + 1]);
      s = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(kk, word(q[0][2 * h], q[0][2 * h + 1]), s, 0, 0, 0);
      lo = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(kk, word(q[1][2 * h], q[1][2 * h + 1]), lo, 0, 0, 0);
    }
    s += lo * 0.0625f;
  }
  return s;
}

// Maximum over the four lanes of a column (lane ^ 16, lane ^ 32, both).
__device__ __forceinline__ float max_xor16_32(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Maximum over a lane and lane ^ 32.
__device__ __forceinline__ float max_xor32(float v) {
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

// cap * tanh(y), off by at most 2^-19 of itself. 1 - 2 / (1 + e^2y) is off by some 2^-21.3 of 1
// everywhere, which is too much of a small y: below 1/2 the series y - y^3 / 3 + 2 y^5 / 15 - ..,
// whose first term left out is 2^-23 of y there, and in fewer cycles.
__device__ __forceinline__ float capped_near(float y, float cap) {
  const float z = y * y;
  float c = fmaf(z, 21844.0f / 6081075.0f, -1382.0f / 155925.0f);
  c = fmaf(z, c, 62.0f / 2835.0f);
  c = fmaf(z, c, -17.0f / 315.0f);
  c = fmaf(z, c, 2.0f / 15.0f);
  c = fmaf(z, c, -1.0f / 3.0f);
  return cap * fmaf(z * c, y, y);
}
__device__ __forceinline__ float capped_any(float y, float cap) {
  const float e = __builtin_amdgcn_exp2f(y * 2.8853900817779268f);  // e^2y; inf: 1
  const float far = cap * fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
  return fabsf(y) < 0.5f ? capped_near(y, cap) : far;
}
// N scores s times mul, capped. Where all of a wave's lie below half the cap, as they mostly do, they
// take the series alone: 23 rows of 1,024 seen keys 21.0 us, 21.5 with both formed for each score.
template <int N, typename T>
__device__ __forceinline__ void cap_scores(T& s, float mul, float cap) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] *= mul;
    most = fmaxf(most, fabsf(s[i]));
  }
  if (__all(most < 0.5f)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = capped_near(s[i], cap);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few registers at once
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = capped_any(s[i], cap);
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
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
  int r, first;  // row and its first item; r = -1: none, and first the items of all rows
  Kv8Row row;
};

// The row that item g lies in, where a row has items(r, row) of them, by the wave.
template <typename F>
__device__ __forceinline__ Found find_row(const Kv8Plan& p, int g, F items) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b = 0; b < p.n; b += 64) {
    const int r = b + lane;
    Kv8Row row = r < p.n ? p.rows[r] : Kv8Row{-1, 0, 0, 0};
    row.fresh = kv8_tokens(p, row);
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
  return Found{-1, before, {-1, 0, 0, 0}};
}

// Zeros for those of the 64 tokens from t0 on whose rows are refused, by `threads` threads.
__device__ __forceinline__ void zero_refused(const Kv8AttnArgs& a, int64_t t0, int tid, int threads) {
  const int64_t mine = t0 + (threadIdx.x & 63);
  const int quads = a.p.D / 4;
  uint64_t none = __ballot(mine < a.p.T && a.p.tok_row[mine] == -1);
  for (; none; none &= none - 1) {
    const int64_t t = t0 + __ffsll((unsigned long long)none) - 1;
    for (int i = tid; i < a.p.Hq * quads; i += threads)
      *reinterpret_cast<u32x2*>(a.out + t * a.os + (i / quads) * a.ohs + i % quads * 4) = (u32x2){0u, 0u};
  }
}

// 1 / (1 + e^-x), off by some 2^-22 of itself
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// Four outputs of a head from dim on: times sigmoid(gate) where there is one, rounded once.
__device__ __forceinline__ void store4(const Kv8AttnArgs& a, int64_t t, int h, int dim, float* o) {
  if (a.gate) {
    const u32x2 g = *reinterpret_cast<const u32x2*>(a.gate + t * a.gs + h * a.ghs + dim);
    o[0] *= sigmoid(bf_lo(g.x));
    o[1] *= sigmoid(bf_hi(g.x));
    o[2] *= sigmoid(bf_lo(g.y));
    o[3] *= sigmoid(bf_hi(g.y));
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
  Kv8Span span;
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
  x.lo = a.window > 0 ? max(x.cpos - a.window, -1) : -1;  // keys above it
  x.span = kv8_span(x.pos0, x.pos0 + x.nt - 1, a.window, x.pf, x.total);
  return x;
}

// A lane's dims of its column's q, pieces of 16 (piece i from step * i on, pairs of them side by
// side with PAIR) in two e4m3 parts, in turn; returns the exponent of the column. The column
// lies in lanes l, l ^ 32 and, without PAIR, l ^ 16.
template <int N, bool PAIR>
__device__ __forceinline__ int q_pieces(const uint16_t* q, bool valid, u32x4* out) {
  u32x4 x[N][2];
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int at = PAIR ? 64 * (i >> 1) + 16 * (i & 1) : 64 * i;
      x[i][b] = valid ? *reinterpret_cast<const u32x4*>(q + at + 8 * b) : (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t lo = x[i][b][w] & 0x7fffu, hi = (x[i][b][w] >> 16) & 0x7fffu;
        mx = max(mx, max(lo >= 0x7f80u ? 0u : lo, hi >= 0x7f80u ? 0u : hi));
      }
    }
  // bf16 patterns are in the order of their sizes, and so are they as f32
  const float size = __uint_as_float(mx << 16);
  const uint32_t bits = __float_as_uint(PAIR ? max_xor32(size) : max_xor16_32(size));
  // the least e with the largest <= 448 * 2^e (448 = 1.75 * 2^8)
  const int e = max((int)(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -100);
  const float inv = pow2(-e);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u32x4 hi, lo;
#pragma unroll
    for (int w = 0; w < 4; ++w) {  // 4 dims a word
      const uint32_t a = x[i][w >> 1][2 * (w & 1)], b = x[i][w >> 1][2 * (w & 1) + 1];
      const float f[4] = {bf_lo(a) * inv, bf_hi(a) * inv, bf_lo(b) * inv, bf_hi(b) * inv};
      int h = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
      h = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], h, true);
      const float r[4] = {(f[0] - __builtin_amdgcn_cvt_f32_fp8(h, 0)) * 16.f,
                          (f[1] - __builtin_amdgcn_cvt_f32_fp8(h, 1)) * 16.f,
                          (f[2] - __builtin_amdgcn_cvt_f32_fp8(h, 2)) * 16.f,
                          (f[3] - __builtin_amdgcn_cvt_f32_fp8(h, 3)) * 16.f};
      int l = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
      l = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], l, true);
      hi[w] = (uint32_t)h;
      lo[w] = (uint32_t)l;
    }
    out[2 * i] = hi;
    out[2 * i + 1] = lo;
  }
  return e;
}
// of 16 columns: dims 64 i + 16 g4 ..; of 32: dims 64 i + 32 hf .. (q already moved there)
template <int NK>
__device__ __forceinline__ int q_parts(const uint16_t* q, bool valid, u32x4* out) {
  return q_pieces<NK, false>(q, valid, out);
}
template <int NK>
__device__ __forceinline__ int q_parts32(const uint16_t* q, bool valid, u32x4* out) {
  return q_pieces<2 * NK, true>(q, valid, out);
}

// sc * 2^e; an e that leaves nothing of any score stays a factor, and what has no room in f32 its
// largest number, so that scores of zero stay zero
__device__ __forceinline__ float factor_of(float sc, int e) {
  return __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(sc, max(e, -110)), -FLT_MAX, FLT_MAX);
}

// Bits of those of a lane's `count` scores whose keys lie below n, four keys side by side every
// STEP from 0 on.
template <int STEP>
__device__ __forceinline__ uint32_t first_scores(int n, int count) {
  const int k = min(max(n, 0), STEP * count / 4);
  return (1u << (4 * (k / STEP) + min(k % STEP, 4))) - 1u;
}

// The running softmax of 16 columns over blocks of 32 keys: lane (g4, c) holds keys 4 g4 + r and
// 16 + 4 g4 + r of a block for column c, and dims 16 d + 4 g4 + r of its outputs in units of
// 2^(unit - kUnit).
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

  // Scores S of the block at key0 to weights P; e: the exponent of its keys and q, ev: of its values
  __device__ __forceinline__ u32x4 weights(const f32x4* S, const Score& sc, const Group& x, int key0,
                                           int e, int ev, uint32_t& seen) {
    const int g4 = (threadIdx.x & 63) >> 4;
    float s[8];
    const float mul = factor_of(sc.mul, e);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = S[i >> 2][i & 3];
    const int k0 = key0 + 4 * g4;  // score i is of key k0 + 16 (i / 4) + i % 4
    if (__builtin_expect(sc.cap > 0.f, 0)) {
      asm volatile("");  // a branch: the caps are many instructions
      cap_scores<8>(s, mul, sc.cap);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] *= mul;
    }
    if (__builtin_expect(sc.sloped, 0)) {
      asm volatile("");
      const float far = sc.slope * (float)(k0 - x.cpos);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += fmaf(sc.slope, (float)(16 * (i >> 2) + (i & 3)), far);
    }
    seen = 0xffu;
    // wave-uniform: every token of the group sees every key of the block
    const bool all = (key0 + kBlock - 1 <= x.pos0 && key0 > x.pos0 + x.nt - 1 - sc.window) ||
                     key0 + kBlock <= x.pf;
    if (__builtin_expect(!all, 0)) {
      asm volatile("");
      auto below = [](int n) { return first_scores<16>(n, 8); };  // of keys below k0 + n
      seen = (below(x.cpos + 1 - k0) & ~below(x.lo + 1 - k0)) | below(x.valid ? x.pf - k0 : 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = (seen >> i) & 1u ? s[i] : -INFINITY;
    }
    float bm = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                     fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    bm = max_xor16_32(bm);
    // m follows the maximum once it is passed by 2^kStep: weights are at most that
    if (__builtin_expect(__any(bm > m + kStep) || !unit_holds(ev, unit), 0)) {
      const float mn = fmaxf(m, bm);
      float corr = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;  // m = -inf: 0
      m = mn;
      l *= corr;
      if (!unit_holds(ev, unit)) {
        corr = __builtin_amdgcn_ldexpf(corr, unit - ev);
        unit = ev;
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) O[d] *= corr;
    }
    const int up = kUnit + ev - unit;
    const float mref = (m == -INFINITY ? 0.f : m) - (float)up;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = __builtin_amdgcn_exp2f(s[i] - mref);
    const u32x4 P = {pk_f16(s[0], s[1]), pk_f16(s[2], s[3]), pk_f16(s[4], s[5]), pk_f16(s[6], s[7])};
    l = fmaf(add_f16(P[2], add_f16(P[0], 0.f)) + add_f16(P[3], add_f16(P[1], 0.f)), pow2(-up), l);
    return P;
  }

  // O += the block's values (raw bytes v, as loaded) . P. `total`: the row's keys.
  __device__ __forceinline__ void values(u32x4* v, u32x4 P, int key0, int total, bool has_nan,
                                         uint32_t seen) {
    if (__builtin_expect(key0 + kBlock > total, 0)) {  // keys past the row's end may hold anything
      const int g4 = (threadIdx.x & 63) >> 4;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = total - key0 - 4 * ((g4 & 1) + 2 * (w >> 1) + 4 * (w & 1));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) v[i][w] = first_keys(v[i][w], n);
      }
    }
    if (__builtin_expect(has_nan, 0)) {
      // NaN values leave the product; a column that sees one of their keys gets a NaN sum
      u32x4 keys = {0u, 0u, 0u, 0u};  // top bits of the bytes of keys with a NaN in the lane's dims
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t top = ((v[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          v[i][w] &= ~((top >> 7) * 0xffu);
          keys[w] |= top;
        }
      const int g4 = (threadIdx.x & 63) >> 4;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) keys[w] |= __shfl_xor(keys[w], off, 64);
        keys[w] |= __shfl_xor(keys[w], 32, 64);  // the other 16 dims, same keys
      }
      const uint32_t k0 = g4 & 2 ? keys[2] : keys[0], k1 = g4 & 2 ? keys[3] : keys[1];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (((seen >> i) & 1u & (k0 >> (8 * i + 7))) | ((seen >> (4 + i)) & 1u & (k1 >> (8 * i + 7))))
          l = __builtin_nanf("");
    }
    const f16x8 ph = __builtin_bit_cast(f16x8, P);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      u32x2 va, vb;
      v_operands(v[i], va, vb);
      O[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(to_f16(va.x, va.y), ph, O[2 * i], 0, 0, 0);
      O[2 * i + 1] =
          __builtin_amdgcn_mfma_f32_16x16x32_f16(to_f16(vb.x, vb.y), ph, O[2 * i + 1], 0, 0, 0);
    }
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

// Items of a row of few tokens: (group, kv head, chunk) in this order. Whole pages for each of a
// chunk's waves.
__device__ __forceinline__ Kv8Cut chunks_of(const Kv8AttnArgs& a, const Kv8Row& row, int r, int tpg) {
  if (row.fresh <= 0) return Kv8Cut{0, 1, 0};
  const int total = row.pos + row.fresh;
  const int pf = a.prefix ? min(max(a.prefix[r], 0), total) : 0;
  return kv8_cut(row.pos, row.fresh, a.window, pf, tpg,
                 kv8_chunks(a.p.n, a.p.Hkv, (row.fresh + tpg - 1) / tpg),
                 kv8_chunk_waves(a.p.n, a.p.Hkv), 1);
}

// Items of a row in a step of tiles: (tile from the last one on, split). By row alone where pages
// are cut, and by the step's bounds, which rows of fewer than kKv8TileTokens tokens have their own
// of: they are few tiles with as many pages as any.
__device__ __forceinline__ Kv8Cut splits_of(const Kv8AttnArgs& a, const Kv8Row& row, int r, int tpt,
                                            const Kv8Splits& most_splits) {
  if (row.fresh <= 0) return Kv8Cut{0, 1, 0};
  const int pieces = row.fresh < kKv8TileTokens ? most_splits.few : most_splits.many;
  if (pieces <= 1) return Kv8Cut{(row.fresh + tpt - 1) / tpt, 1, 1};
  const int total = row.pos + row.fresh;
  const int pf = a.prefix ? min(max(a.prefix[r], 0), total) : 0;
  return kv8_cut(row.pos, row.fresh, a.window, pf, tpt, pieces, 1, kSplitPages);
}
// Partial results of a tile's splits: 128 columns of D + 4 floats each
template <int D>
__device__ __forceinline__ float* split_part(const Kv8Plan& p, float* part, const Kv8Splits& most, int r,
                                             int fresh, int tile, int j) {
  constexpr size_t kStride = (size_t)32 * kKv8TileWaves * (D + 4);
  if (fresh >= kKv8TileTokens)
    return part + ((size_t)(p.tiles[r] + tile) * p.Hkv + j) * most.many * kStride;
  const size_t at = (size_t)r * kv8_few_tiles(p.Hq / p.Hkv) + tile;
  return part + (kv8_tile_groups(D) + (at * p.Hkv + j) * most.few) * kStride;
}

}  // namespace

// Work-group g takes the chunks g, g + grid, ... of all rows' items; its W waves every W-th page
// of a chunk each, and they join in LDS: one partial a chunk. A wave loads the next page's
// keys as soon as this page's scores are formed, its values after this page's products: 32 KiB of
// 256 dims in flight for each wave, which takes 512 registers and so a SIMD. Bound by HBM: 64
// rows at 4,096 keys (279 MB of pages, 2 kv heads of 256 dims) 56 us, 5.0 TB/s where a large copy
// reaches 5.2; 23 rows that see 1,024 keys each (49 MB, 8 of 128, capped) 15.0 us. Bound by latency where
// a wave has a page or none: a row at 32,768 keys (34 MB) 15 us.
template <int D, int W>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void attn8_chunk_kernel(Kv8AttnArgs a, float* __restrict__ part) {
  constexpr int NK = D / 64, DB = D / 16;
  __shared__ u32x4 qlds[2 * NK][64];
  __shared__ f32x4 os[W > 1 ? W : 1][W > 1 ? 16 : 1][D / 4];  // each wave's outputs: column, dims
  __shared__ float ms[W][16], ls[W][16];
  const Kv8Plan& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.Hq / p.Hkv, tpg = 16 / G, row_parts = kv8_row_parts(p.n, p.Hkv) * p.Hkv;
  auto items = [&](int r, const Kv8Row& row) {
    const Kv8Cut k = chunks_of(a, row, r, tpg);
    return k.items * k.n * p.Hkv;
  };
  for (int g = blockIdx.x;; g += gridDim.x) {
    const Found f = find_row(p, g, items);
    if (f.r < 0) break;
    const Kv8Cut ch = chunks_of(a, f.row, f.r, tpg);
    const int local = g - f.first, seg = local / ch.n, chunk = local - seg * ch.n;
    const int grp = seg / p.Hkv, j = seg - grp * p.Hkv;
    const Group x = group_of(a, f.row, f.r, grp, j, G, tpg, c);
    const Score sc = score_of(a, x);
    const int v1 = kv8_piece_end(ch, chunk, x.span.count());
    if (W > 1 && g != (int)blockIdx.x) __syncthreads();  // the chunk before is written out
    int eq;  // every wave forms q: its exponent is in registers
    {
      u32x4 q[2 * NK];
      eq = q_parts<NK>(a.q + x.t * a.qs + x.h * a.qhs + 16 * g4, x.valid, q);
      if (w == 0) {
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i) qlds[i][lane] = q[i];
      }
    }
    const int32_t* const trow = p.table + (size_t)f.row.slot * p.max_pages;
    // ids and exponents of 64 of the chunk's pages, one a lane
    int vbase = chunk * ch.cp, pid = 0, eks = 0, evs = 0;
    auto ids = [&](int v) {
      vbase = v;
      pid = v + lane < v1 ? trow[x.span.page(v + lane)] : 0;
      const int32_t* const e = a.exps + (size_t)pid * 2 * p.Hkv + j;
      eks = e[0];
      evs = e[p.Hkv];
      // waited for here: a wait behind the branch that reloads them would be one for every
      // page load in flight, taken or not
      asm volatile("" ::"v"(pid), "v"(eks), "v"(evs));
    };
    const uint8_t* const base = a.pages + (size_t)j * (kPage * D);
    const size_t page_bytes = (size_t)2 * p.Hkv * kPage * D, v_shift = (size_t)p.Hkv * kPage * D;
    // a page's halves of 32 keys, 32 * D contiguous bytes each of K and V
    u32x4 kf[2][2 * NK], vf[2][DB / 2];
    auto page_of = [&](int v) {
      return base + (size_t)(uint32_t)__builtin_amdgcn_readlane(pid, v - vbase) * page_bytes;
    };
    auto load = [&](const uint8_t* s, u32x4(&f)[DB / 2]) {
#pragma unroll
      for (int i = 0; i < DB / 2; ++i)
        f[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(s) + i * 64 + lane);
    };
    constexpr int kHalf = kBlock * D;
    Online<D> on;
    on.clear();
    ids(vbase);
    int v = vbase + w;
    if (v < v1) {
      const uint8_t* const cur = page_of(v);
      load(cur, kf[0]);
      load(cur + v_shift, vf[0]);
      load(cur + kHalf, kf[1]);
      load(cur + v_shift + kHalf, vf[1]);
    }
    lds_barrier();  // q
    // page v, with the loads of the wave's next one behind its products; the last page (a call
    // of its own) has none to issue: loads under a branch would be waited for as a whole
    auto page = [&](auto lastc) {
      constexpr bool last = decltype(lastc)::value;
      const int key0 = x.span.page(v) * kPage;
      const int ek = (int)(int8_t)__builtin_amdgcn_readlane(eks, v - vbase);
      const int wv = __builtin_amdgcn_readlane(evs, v - vbase), ev = (int)(int8_t)wv;
      const uint8_t* nxt = nullptr;
      if constexpr (!last) {
        if (v + W - vbase >= 64) ids(v + W);
        nxt = page_of(v + W);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        asm volatile("" ::: "memory");  // q is re-read from LDS for every block
        f32x4 S[2];
        {
          u32x4 q[2 * NK];
#pragma unroll
          for (int i = 0; i < 2 * NK; ++i) q[i] = qlds[i][lane];
          S[0] = scores16<NK>(kf[h], q);
          S[1] = scores16<NK>(kf[h] + NK, q);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!last) load(nxt + h * kHalf, kf[h]);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t seen;
        const u32x4 P = on.weights(S, sc, x, key0 + kBlock * h, eq + ek, ev, seen);
        on.values(vf[h], P, key0 + kBlock * h, x.total, (wv & kNanFlag) != 0, seen);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!last) load(nxt + v_shift + h * kHalf, vf[h]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (v < v1) {
      for (; v + W < v1; v += W) page(std::false_type{});
      page(std::true_type{});
    }
    float* const out = part + ((size_t)f.r * row_parts + seg * ch.n + chunk) * 16 * (D + 4);
    const float lw = on.sum();
    if constexpr (W == 1) {
      if (!x.valid) continue;
      if (ch.n == 1) {
        const float inv = __builtin_amdgcn_ldexpf(1.0f / lw, on.unit - kUnit);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          float o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = on.O[d][r] * inv;
          store4(a, x.t, x.h, 16 * d + 4 * g4, o);
        }
      } else {
        float* const pr = out + c * (D + 4);
        if (g4 == 0) {
          pr[0] = on.m;
          pr[1] = lw;
        }
        const float one = __builtin_amdgcn_ldexpf(1.0f, on.unit - kUnit);
#pragma unroll
        for (int d = 0; d < DB; ++d)
          *reinterpret_cast<f32x4*>(pr + 4 + 16 * d + 4 * g4) = on.O[d] * one;
      }
      continue;
    }
    // the waves' results under their common maximum
    if (g4 == 0) ms[w][c] = on.m;
    lds_barrier();
    float M = ms[0][c];
#pragma unroll
    for (int i = 1; i < W; ++i) M = fmaxf(M, ms[i][c]);
    const float fac = on.m == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : exp2f(on.m - M);
    if (g4 == 0) ls[w][c] = lw * fac;
    const float fo = __builtin_amdgcn_ldexpf(fac, on.unit - kUnit);
    if (x.valid) {
#pragma unroll
      for (int d = 0; d < DB; ++d) os[w][c][4 * d + g4] = on.O[d] * fo;
    }
    lds_barrier();
    const int cols = x.nt * G;
    for (int i = tid; i < cols * (D / 4); i += 64 * W) {
      const int col = i / (D / 4), d = i - col * (D / 4);
      float l = ls[0][col], m = ms[0][col];
      f32x4 o = os[0][col][d];
#pragma unroll
      for (int k = 1; k < W; ++k) {
        l += ls[k][col];
        m = fmaxf(m, ms[k][col]);
        o += os[k][col][d];
      }
      if (ch.n == 1) {
        o *= 1.0f / l;
        const int tok = col / G;
        float of[4] = {o[0], o[1], o[2], o[3]};
        store4(a, (int64_t)f.row.cu + grp * tpg + tok, j * G + col - tok * G, 4 * d, of);
      } else {
        float* const pr = out + (size_t)col * (D + 4);
        *reinterpret_cast<f32x4*>(pr + 4 + 4 * d) = o;
        if (d == 0) {
          pr[0] = m;
          pr[1] = l;
        }
      }
    }
  }
  // tokens of refused rows: zeros, each work-group its share of the step's
  for (int64_t t0 = blockIdx.x * 64; t0 < p.T; t0 += gridDim.x * 64) zero_refused(a, t0, tid, 64 * W);
}

// Rows of few tokens: grid (n * per, Hq), block 64 W; token k < per of row r, a head: its chunks,
// chunk i in sum i % 16, wave w the sums w, w + W, ..; then the sums in order. Rows of a single
// chunk are written already. Bound by latency, the row, its chunks and their rows one after the
// other: 4 waves with four sums each take a token's 128 chunks of 16 heads of 256 dims in 6 us,
// 16 waves with one sum each, which a work-group has to wait for, in 7.5.
template <int D>
__global__ __launch_bounds__(256) void attn8_join_kernel(Kv8AttnArgs a, const float* __restrict__ part,
                                                         int per) {
  constexpr int W = 4, DPL = D / 64, kPer = 16 / W;
  constexpr size_t kStride = (size_t)16 * (D + 4);  // of a token's chunks
  typedef float fvec __attribute__((ext_vector_type(DPL)));
  __shared__ float sum[16][D];
  const Kv8Plan& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = blockIdx.x / per, k = blockIdx.x - r * per;
  const Kv8Row row = p.rows[r];
  if (k >= kv8_tokens(p, row)) return;
  const int G = p.Hq / p.Hkv, tpg = 16 / G, j = h / G, grp = k / tpg, c = (k - grp * tpg) * G + h - j * G;
  const int nch = chunks_of(a, row, r, tpg).n;
  if (nch < 2) return;
  const int64_t t = (int64_t)row.cu + k;
  const float* const pc =
      part + ((size_t)(r * kv8_row_parts(p.n, p.Hkv) + grp * nch) * p.Hkv + j * nch) * kStride + c * (D + 4);
  // 64 chunks' rows go out before their maxima and sums, one a lane, are waited for
  fvec v[4][kPer];
  auto rows = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (b + 16 * q < nch) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          v[q][i] = *reinterpret_cast<const fvec*>(
              pc + min(b + 16 * q + wave + W * i, nch - 1) * kStride + 4 + DPL * lane);
      }
  };
  rows(0);
  float mi = lane < nch ? pc[lane * kStride] : -INFINITY;
  float li = lane < nch ? pc[lane * kStride + 1] : 0.f;
  float M = mi;
  for (int i = lane + 64; i < nch; i += 64) M = fmaxf(M, pc[i * kStride]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  if (M == -INFINITY) M = 0.f;  // NaN scores alone
  float L = 0.f;
  fvec A[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) A[i] = (fvec)(0.f);
  for (int b = 0; b < nch; b += 64) {
    if (b) {
      rows(b);
      mi = b + lane < nch ? pc[(b + lane) * kStride] : -INFINITY;
      li = b + lane < nch ? pc[(b + lane) * kStride + 1] : 0.f;
    }
    const float wi = exp2f(mi - M);
    L += li != 0.f ? wi * li : 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (b + 16 * q < nch) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int l = 16 * q + wave + W * i;
          const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wi), l));
          const float s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(li), l));
          if (s != 0.f) A[i] += v[q][i] * f;  // chunks without a visible key hold nothing
        }
      }
  }
  L = wave_sum(L);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
#pragma unroll
    for (int d = 0; d < DPL; ++d) sum[wave + W * i][DPL * lane + d] = A[i][d];
  __syncthreads();
  if (tid < D / 4) {
    const float inv = 1.0f / L;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) s += *reinterpret_cast<const f32x4*>(&sum[i][4 * tid]);
    float o[4] = {s[0] * inv, s[1] * inv, s[2] * inv, s[3] * inv};
    store4(a, t, h, 4 * tid, o);
  }
}

// Tiles whose pages are split: grid (those of rows of few tokens, if any may be split, then those
// of the others, if any may, Hkv, kKv8TileWaves), block 256: a wave's 32 columns by eights, 8 lanes for
// every fourth split of each, those in order and then the four sums. Bound by latency, the row and
// its pieces' rows one after the other: 2,268 tokens of 16 heads of 64 dims, 3 pieces each (30 MB),
// 14 us; with the maxima and the sums in two passes 17, by 32 dims a work-group 19.
template <int D>
__global__ __launch_bounds__(256) void attn8_join_tiles_kernel(Kv8AttnArgs a, float* __restrict__ part,
                                                               Kv8Splits most_splits) {
  constexpr size_t kStride = (size_t)32 * kKv8TileWaves * (D + 4);
  const Kv8Plan& p = a.p;
  const int G = p.Hq / p.Hkv, tpw = 32 / G, tpt = kKv8TileWaves * tpw, j = blockIdx.y;
  const int ft = kv8_few_tiles(G), few = most_splits.few > 1 ? p.n * ft : 0;
  int r, tile;
  Kv8Row row;
  if ((int)blockIdx.x < few) {
    r = blockIdx.x / ft;
    tile = blockIdx.x - r * ft;
    row = p.rows[r];
    row.fresh = kv8_tokens(p, row);
    if (row.fresh >= kKv8TileTokens) return;
  } else {
    const Found f = find_row(p, blockIdx.x - few, [&](int, const Kv8Row& x) {
      return x.fresh >= kKv8TileTokens ? (x.fresh + tpt - 1) / tpt : 0;
    });
    if (f.r < 0) return;
    r = f.r;
    tile = blockIdx.x - few - f.first;
    row = f.row;
  }
  const int n = splits_of(a, row, r, tpt, most_splits).n;
  if (n < 2) return;
  const int wave = blockIdx.z;
  const int dim = 4 * (threadIdx.x & 7);  // and those 32, 64, .. further on
  const int g = (threadIdx.x >> 3) & 3;
  const float* const base = split_part<D>(p, part, most_splits, r, row.fresh, tile, j);
  auto over_four = [](float x, auto join) {
    x = join(x, __shfl_xor(x, 8, 64));
    return join(x, __shfl_xor(x, 16, 64));
  };
  auto add = [](float x, float y) { return x + y; };
#pragma nounroll
  for (int c = threadIdx.x >> 5; c < 32; c += 8) {
    const int ctok = c / G, tok = tile * tpt + wave * tpw + ctok;
    if (ctok >= tpw || tok >= row.fresh) return;  // and so are those behind it
    const float* const pc = base + (size_t)(wave * 32 + c) * (D + 4);
    float M = -INFINITY, L = 0.f;
    f32x4 A[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) A[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // the sums so far times 2^(M - to) as the maximum goes on to `to`; NaN scores alone leave it
    auto rise = [&](float to) {
      const float f = exp2f(M - (to == -INFINITY ? 0.f : to));
      L *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) A[i] *= f;
      M = to;
    };
#pragma unroll(512 / D)
    for (int s = g; s < n; s += 4) {
      const float m = pc[s * kStride], l = pc[s * kStride + 1];
      f32x4 v[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) v[i] = *reinterpret_cast<const f32x4*>(pc + s * kStride + 4 + dim + 32 * i);
      if (l == 0.f) continue;  // a split without a visible key holds nothing
      rise(fmaxf(M, m));
      const float f = exp2f(m - (M == -INFINITY ? 0.f : M));
      L += f * l;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) A[i] += v[i] * f;
    }
    rise(over_four(M, [](float x, float y) { return fmaxf(x, y); }));
    const float inv = 1.0f / over_four(L, add);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      float o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = over_four(A[i][k], add) * inv;
      if (i % 4 == g) store4(a, (int64_t)row.cu + tok, j * G + c - ctok * G, dim + 32 * i, o);
    }
  }
}

// Prompts. Work-group (tile, kv head): a tile is NW * (32 / G) consecutive tokens of a row, wave w
// takes 32 / G of them from w (32 / G) on; the (token, query head) pairs are its 32 columns. A page
// of K and V is copied into LDS by DMA a page ahead, two buffers of each, and read by all waves.
// Rows of the products are 32 keys or dims, so that an operand read from LDS, and a value's
// conversion, serves 32 columns.
//
// Lane (hf, c), hf = lane / 32, holds keys 8 i + 4 hf + r of a block of 32 (i, r = 0 .. 3) for
// column c, and dims 32 t + 8 i + 4 hf + r of its outputs in units of 2^(unit - kUnit).
//
// As many waves a SIMD as the outputs and q's parts (128 + 64 registers at D = 256) leave room for,
// 2, 3 and 4 at 256, 128 and 64 dims; one's products run beside the others' softmax, so that a
// wave's own steps stay in order. 8,192 tokens of 16 query heads over 2 of 256 dims: one wave a
// SIMD with the steps of two blocks side by side 665 us, two 483 (483 to 523 by box); products and softmax of half
// the waves in turn, by barriers, were as fast (508, where the rest took 500). At that rate (1.1
// PFLOP/s, a quarter of the matrix time on top for the scores' second part) the clock, not a unit,
// is what gives: the f16 products alone run at 1.6 GHz on such numbers, and at 2.2 on constants.
// 19 rows of 1 .. 571 tokens of 32 query heads over 8 of 128 dims: 255 us in two waves a SIMD, 231
// in three.
template <int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 256 ? 2 : D == 128 ? 3 : 4) void attn8_tile_kernel(
    Kv8AttnArgs a, float* __restrict__ part, Kv8Splits most_splits) {
  constexpr int NK = D / 64, NT = D / 32, kTile16 = kPage * D / 16;  // 16-byte pieces of a tile
  constexpr int kLoads = kTile16 / 64 / NW;                          // of a wave for a tile
  static_assert(kTile16 % (64 * NW) == 0, "whole pieces for each wave");
  __shared__ u32x4 lk0[kTile16], lk1[kTile16], lv0[kTile16], lv1[kTile16];
  // a lane's column: its position (-1: none), its slope, the exponent of its q
  struct Column { int pos; float slope; int eq, pad; };
  __shared__ Column columns[D == 256 ? 64 * NW : 1];
  const Kv8Plan& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, hf = lane >> 5, c = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.Hq / p.Hkv, tpw = 32 / G, tpt = NW * tpw, j = blockIdx.y;
  const Found f = find_row(p, blockIdx.x, [&](int r, const Kv8Row& row) {
    const Kv8Cut s = splits_of(a, row, r, tpt, most_splits);
    return s.items * s.n;
  });
  if (f.r < 0) {  // a work-group to spare (the last one is): tokens of refused rows, zeros
    const int first = ((int)(blockIdx.x - f.first) * gridDim.y + j) * NW + w;
    const int step = ((int)gridDim.x - f.first) * gridDim.y * NW;
    for (int64_t t0 = (int64_t)first * 64; t0 < p.T; t0 += (int64_t)step * 64)
      zero_refused(a, t0, lane, 64);
    return;
  }
  const Kv8Row row = f.row;
  const Kv8Cut sp = splits_of(a, row, f.r, tpt, most_splits);
  const int local = blockIdx.x - f.first, split = local % sp.n;
  const int tile = sp.items - 1 - local / sp.n;  // longest first
  const int total = row.pos + row.fresh;
  const int pf = a.prefix ? min(max(a.prefix[f.r], 0), total) : 0;
  const int p0 = row.pos + tile * tpt;  // the tile's first position
  const Kv8Span span = kv8_span(p0, min(p0 + tpt, total) - 1, a.window, pf, total);
  const int v0 = split * sp.cp;
  const int count = kv8_piece_end(sp, split, span.count());  // pages [v0, count)
  // the tile's partial results, if its pages are split: columns (wave, c)
  float* const out = split_part<D>(p, part, most_splits, f.r, row.fresh, tile, j) +
                     (size_t)split * (32 * NW * (D + 4));
  if (v0 >= count) {  // nothing in this split (the tile sees fewer pages than others)
    for (int i = tid; i < 32 * NW; i += 64 * NW) {
      out[(size_t)i * (D + 4)] = -INFINITY;
      out[(size_t)i * (D + 4) + 1] = 0.f;
    }
    return;
  }
  // the wave's positions
  const int w0 = p0 + w * tpw, wn = min(max(total - w0, 0), tpw);
  const int window = a.window > 0 ? a.window : INT32_MAX / 2;
  const float sm = __int_as_float(__builtin_amdgcn_readfirstlane(
      __float_as_int(a.softcap > 0.f ? a.scale / a.softcap : a.scale * 1.4426950408889634f)));
  const int32_t* const trow = p.table + (size_t)row.slot * p.max_pages;
  int vbase = 0, pid = 0, eks = 0, evs = 0;
  auto ids = [&](int v) __attribute__((always_inline)) {
    vbase = v;
    pid = v + lane < count ? trow[span.page(v + lane)] : 0;
    const int32_t* const e = a.exps + (size_t)pid * 2 * p.Hkv + j;
    eks = e[0];
    evs = e[p.Hkv];
    asm volatile("" ::"v"(pid), "v"(eks), "v"(evs));
  };
  ids(v0);
  const uint8_t* const base = a.pages + (size_t)j * (kPage * D);
  const size_t page_bytes = (size_t)2 * p.Hkv * kPage * D, v_shift = (size_t)p.Hkv * kPage * D;
  auto page_of = [&](int v) __attribute__((always_inline)) {
    uint64_t at = (uint64_t)base +
                  (size_t)(uint32_t)__builtin_amdgcn_readlane(pid, min(v, count - 1) - vbase) * page_bytes;
    asm("" : "+s"(at));  // lanes add their 32-bit offsets to it
    return reinterpret_cast<const uint8_t*>(at);
  };
  // K or V of page v into a buffer: a wave copies its share of the 1 KiB pieces
  auto copy = [&](int v, u32x4* dst, size_t shift) __attribute__((always_inline)) {
    const uint8_t* const src = page_of(v) + shift + w * (kLoads * 1024);
    const uint32_t mine = lane * 16;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds(
          (const void __attribute__((address_space(1)))*)(src + i * 1024 + mine),
          (void __attribute__((address_space(3)))*)(dst + (w * kLoads + i) * 64), 16, 0, 0);
  };
  copy(v0, lk0, 0);
  copy(v0, lv0, v_shift);
  copy(v0 + 1, lk1, 0);
  copy(v0 + 1, lv1, v_shift);

  // q: dims 64 i + 32 hf .. + 31 of column c, in two e4m3 parts
  u32x4 qh[2 * NK], ql[2 * NK];
  Column mine;
  {
    const int ctok = c / G, h = j * G + c - ctok * G;
    const bool valid = ctok < wn;
    const int64_t t = (int64_t)row.cu + (valid ? w0 + ctok - row.pos : 0);
    u32x4 q[4 * NK];
    const int eq = q_parts32<NK>(a.q + t * a.qs + h * a.qhs + 32 * hf, valid, q);
#pragma unroll
    for (int i = 0; i < 2 * NK; ++i) {
      qh[i] = q[2 * i];
      ql[i] = q[2 * i + 1];
    }
    mine = Column{valid ? w0 + ctok : -1,
                          a.slopes && valid ? a.slopes[h] * 1.4426950408889634f : 0.f, eq, 0};
    if constexpr (D == 256) columns[tid] = mine;
  }
  // at D = 256 from LDS, found anew at each use, which holds no register
  auto column = [&]() __attribute__((always_inline)) {
    if constexpr (D < 256) return mine;
    int at;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(at));
    return columns[64 * w + at];
  };
  // this lane's pieces: of key c of 32 (NK KiB for 16 keys), and of dim c of 32
  const int kat = (c >> 4) * NK * 64 + 32 * hf + (c & 15);
  const int vat = (c >> 4) * 32 + 16 * hf + (c & 15);

  // A distance term can start the accumulators, divided by mk, but for a part that is the lane's:
  // half the work of adding it to the scores (19 ragged rows of 64 dims 102 us, and 97). Not where
  // a cap comes before it, nor beyond the sizes for which the quotient is an f32 number, with mk's
  // power of two 2^-60 at least; and not with more dims, whose registers it has no room in.
  const bool tilt = D == 64 && a.slopes && a.softcap == 0.f && sm >= 0x1p-40f && sm <= 0x1p40f &&
                    __all(fabsf(column().slope) <= 0x1p20f);
  // Nor may masked scores, -inf, meet an mk that is not positive: factor_of()'s 2^-110 of a small
  // scale is none any more, where zero queries meet a page of zeros.
  const bool odd = a.softcap > 0.f || (a.slopes && !tilt) || !(tilt || sm >= 0x1p-16f);
  float m = -INFINITY, l = 0.f, mk, far = 0.f;
  uint32_t seen;
  int unit = 0;
  f32x16 O[NT], S;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[i][r] = 0.f;

  auto both = [](u32x4 x, u32x4 y) __attribute__((always_inline)) {
    return (i32x8){(int)x[0], (int)x[1], (int)x[2], (int)x[3],
                   (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
  };
  // S: scores of half hb of the page in lk, fragments read two ahead
  auto scores = [&](const u32x4* lk, int hb, auto start) __attribute__((always_inline)) {
    constexpr int kOne = 0x7f7f7f7f, kLow = 0x7b7b7b7b;  // 2^0 and 2^-4
    auto key = [&](int i) __attribute__((always_inline)) {
      const int at = kat + (2 * hb * NK + i) * 64;
      return both(lk[at], lk[at + 16]);
    };
#pragma unroll
    for (int i = 0; i < 16; ++i) S[i] = start(i);
    i32x8 kk[2] = {key(0), NK > 1 ? key(1) : key(0)};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      S = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kk[i & 1], both(qh[2 * i], qh[2 * i + 1]), S,
                                                          0, 0, 0, kOne, 0, kOne);
      S = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kk[i & 1], both(ql[2 * i], ql[2 * i + 1]), S,
                                                          0, 0, 0, kOne, 0, kLow);
      if (i + 2 < NK) kk[i & 1] = key(i + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // S, mk, far: scores of the block at kb, keys that a column does not see as -inf, are mk * S + far
  auto prepare = [&](int kb) __attribute__((always_inline)) {
    seen = 0xffffu;
    const int kl = kb + 4 * hf;  // score i is of key kl + 8 (i / 4) + i % 4
    if (__builtin_expect(odd, 0)) {
      asm volatile("");  // a branch, as below: rare and long
      const float cap = a.softcap * 1.4426950408889634f;
      if (cap > 0.f) {
        cap_scores<16>(S, mk, cap);
        mk = 1.f;
      }
      // slopes of zero where there are none: a scale that is small or negative comes here too
      const Column col = column();
      const float slope = col.slope, off = slope * (float)(kl - col.pos);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        S[i] = fmaf(S[i], mk, fmaf(slope, (float)(8 * (i >> 2) + (i & 3)), off));
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few registers at once
      }
      mk = 1.f;
    }
    const bool all = (kb + kBlock - 1 <= w0 && kb > w0 + wn - 1 - window) || kb + kBlock <= pf;
    if (__builtin_expect(!all, 0)) {
      asm volatile("");
      const int cpos = column().pos;
      auto below = [](int k) { return first_scores<8>(k, 16); };  // of keys below kl + k
      seen = (below(cpos + 1 - kl) & ~below(max(cpos - window, -1) + 1 - kl)) |
             below(cpos >= 0 ? pf - kl : 0);
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = (seen >> i) & 1u ? S[i] : -INFINITY;
    }
  };
  // the running maximum follows once it is passed by 2^kStep; ev: the exponent of the block's values
  auto follow = [&](int ev) __attribute__((always_inline)) {
    float bm = fmaxf(S[0], S[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) bm = fmaxf(bm, S[i]);
    bm = max_xor32(fmaf(bm, mk, far));
    if (__builtin_expect(!unit_holds(ev, unit) || __any(bm > m + kStep), 0)) {
      const int to = unit_holds(ev, unit) ? unit : ev;
      const float mn = fmaxf(m, bm);
      float corr = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;  // m = -inf: 0
      m = mn;
      l *= corr;
      corr = __builtin_amdgcn_ldexpf(corr, unit - to);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        O[i] *= corr;
        __builtin_amdgcn_sched_barrier(0);  // not all of them in registers of their own at once
      }
      unit = to;
    }
  };
  u32x4 P[2];
  auto weights = [&](int ev) __attribute__((always_inline)) {
    const int up = kUnit + ev - unit;
    const float mref = (m == -INFINITY ? 0.f : m) - (float)up - far;
    float e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(S[i], mk, -mref));
    // keys 4 hf + r and 16 + 4 hf + r, then those 8 further on: the order of the values' bytes
    P[0] = (u32x4){pk_f16(e[0], e[1]), pk_f16(e[2], e[3]), pk_f16(e[8], e[9]), pk_f16(e[10], e[11])};
    P[1] = (u32x4){pk_f16(e[4], e[5]), pk_f16(e[6], e[7]), pk_f16(e[12], e[13]), pk_f16(e[14], e[15])};
    asm volatile("" : "+v"(P[0]), "+v"(P[1]));  // here, not behind the branches that follow
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) sum[k] = add_f16(P[k][i], sum[k]);
    l = fmaf(sum[0] + sum[1], pow2(-up), l);
  };
  // O += P V of half hb of the page in lv: fragments are read two ahead (the first two apart) and
  // converted beside the products
  u32x4 vr[2];
  auto values_ahead = [&](const u32x4* lv, int hb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) vr[i] = lv[vat + (hb * (D / 16) + 2 * i) * 32];
  };
  auto values = [&](const u32x4* lv, int hb) __attribute__((always_inline)) {
    f16x8 f0 = to_f16(vr[0][0], vr[0][1]);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      O[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f0, __builtin_bit_cast(f16x8, P[0]), O[i], 0, 0, 0);
      const f16x8 f1 = to_f16(vr[i & 1][2], vr[i & 1][3]);
      if (i + 2 < NT) vr[i & 1] = lv[vat + (hb * (D / 16) + 2 * (i + 2)) * 32];
      __builtin_amdgcn_sched_barrier(0);
      O[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f1, __builtin_bit_cast(f16x8, P[1]), O[i], 0, 0, 0);
      if (i + 1 < NT) f0 = to_f16(vr[(i + 1) & 1][0], vr[(i + 1) & 1][1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Half hb of page v, from kb on, before its product where keys past the row's end may hold
  // anything or some hold NaN: those bytes become zeros in LDS (each wave writes all that it
  // reads, the same as the others), and a column that sees the key of a NaN, read from the page
  // itself, gets a NaN sum.
  auto clean = [&](int v, u32x4* lv, int hb, int kb) __attribute__((always_inline)) {
    const uint8_t* const src = page_of(v) + v_shift;
    u32x4 nan_keys = {0u, 0u, 0u, 0u};
#pragma nounroll
    for (int i = 0; i < NT; ++i) {
      const uint32_t at = vat + (hb * (D / 16) + 2 * i) * 32;
      u32x4 x = *reinterpret_cast<const u32x4*>(src + at * 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // the word's four keys, from 4 (hf + 2 (k / 2) + 4 (k % 2)) on
        const uint32_t y = first_keys(x[k], total - kb - 4 * (hf + 2 * (k >> 1) + 4 * (k & 1)));
        const uint32_t top = ((y & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        nan_keys[k] |= top;
        x[k] = y & ~((top >> 7) * 0xffu);
      }
      lv[at] = x;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) nan_keys[k] |= __shfl_xor(nan_keys[k], off, 64);
#pragma unroll
      for (int q = 0; q < 4; ++q)  // scores 4 (k / 2 + 2 (k % 2)) .. are those keys'
        if ((nan_keys[k] >> (8 * q + 7)) & (seen >> (4 * ((k >> 1) + 2 * (k & 1)) + q)) & 1u)
          l = __builtin_nanf("");
    }
  };
  auto exps_of = [&](int v, int& ek, int& ev, bool& nan) __attribute__((always_inline)) {
    const int at = v - vbase;
    ek = (int)(int8_t)__builtin_amdgcn_readlane(eks, at);
    const int wv = __builtin_amdgcn_readlane(evs, at);
    ev = (int)(int8_t)wv;
    nan = (wv & kNanFlag) != 0;
  };
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the first two pages
  lds_barrier();
  const bool idle = wn == 0;  // no tokens for this wave: copies and barriers only
  // Page v in lk and lv, which has landed; the next page's copies are on their way. Products go
  // before another wave's softmax.
  auto page = [&](int v, u32x4* lk, u32x4* lv) __attribute__((always_inline)) {
    const int key0 = span.page(v) * kPage;
    int ek, ev;
    bool nan;
    exps_of(v, ek, ev, nan);
    if (!idle) {
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        const int kb = key0 + hb * kBlock;
        __builtin_amdgcn_s_setprio(1);
        if (__builtin_expect(tilt, 0)) {
          const Column col = column();
          mk = __builtin_amdgcn_ldexpf(sm, max(col.eq + ek, -60));
          far = col.slope * (float)(kb + 4 * hf - col.pos);
          const float part = col.slope * __builtin_amdgcn_rcpf(mk);
          scores(lk, hb, [&](int i) { return part * (float)(8 * (i >> 2) + (i & 3)); });
        } else {
          scores(lk, hb, [](int) { return 0.f; });
          mk = factor_of(sm, column().eq + ek);
        }
        __builtin_amdgcn_s_setprio(0);
        prepare(kb);
        follow(ev);
        values_ahead(lv, hb);
        weights(ev);
        if (__builtin_expect(nan || kb + kBlock > total, 0)) {
          clean(v, lv, hb, kb);
          values_ahead(lv, hb);
        }
        __builtin_amdgcn_s_setprio(1);
        values(lv, hb);
        __builtin_amdgcn_s_setprio(0);
      }
    }
    // the next page has landed everywhere, and no wave reads this one any more
    __builtin_amdgcn_s_waitcnt(0x0F70);
    lds_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "global");
    if (min(v + 2, count - 1) - vbase >= 64) ids(v);
    copy(v + 2, lk, 0);
    copy(v + 2, lv, v_shift);
    __builtin_amdgcn_sched_barrier(0);
  };
  int v = v0;
#pragma nounroll
  for (; v + 2 <= count; v += 2) {
    page(v, lk0, lv0);
    page(v + 1, lk1, lv1);
  }
  if (v < count) page(v, lk0, lv0);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // the last copies (repeats) land before the LDS is given back
  l += __shfl_xor(l, 32, 64);
  const int cpos = column().pos;
  if (cpos < 0) return;
  if (sp.n > 1) {
    float* const pr = out + (size_t)(w * 32 + c) * (D + 4);
    if (hf == 0) {
      pr[0] = m;
      pr[1] = l;
    }
    const float one = __builtin_amdgcn_ldexpf(1.0f, unit - kUnit);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(pr + 4 + 32 * i + 8 * g + 4 * hf) =
            (f32x4){O[i][4 * g], O[i][4 * g + 1], O[i][4 * g + 2], O[i][4 * g + 3]} * one;
    return;
  }
  const int64_t t = (int64_t)row.cu + cpos - row.pos;
  const int h = j * G + c - (cpos - w0) * G;
  const float inv = __builtin_amdgcn_ldexpf(1.0f / l, unit - kUnit);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = O[i][4 * g + r] * inv;
      store4(a, t, h, 32 * i + 8 * g + 4 * hf, o);
    }
}

// Partials of the chunks: all rows' and kv heads' kv8_row_parts()
static size_t chunk_floats(int D) { return (size_t)kKv8Waves * 16 * (D + 4); }

size_t kv8_attn_workspace_bytes(const gdn_kv8_desc& d) {
  // tiles times splits, where there is more than one, are kv8_tile_groups() or less, of the rows
  // of few tokens as of the others
  const size_t tiles = (size_t)2 * kv8_tile_groups(d.head_dim) * 32 * kKv8TileWaves * (d.head_dim + 4);
  return (chunk_floats(d.head_dim) + tiles) * sizeof(float);
}

// Pieces that the pages of at most `tiles` work-groups are cut into. Two lie on a CU side by side
// (D = 64: four): tiles for half of the places or fewer are cut to fill them, 1,024 tokens behind
// 4,096 (D = 256, 130 tiles) 117 us in 3 pieces and 148 in 5; more tiles into two rounds of work,
// 19 ragged rows (D = 256, 320 at most) 268 us whole and 209 in 3; those of 64 dims (356) 107 us in
// 2 pieces, 93 in 3, 94 in 5.
static int tile_pieces(int64_t tiles, int D) {
  return max(1, (int)((D == 64 ? 1280 : tiles <= 256 ? 512 : 1024) / tiles));
}

template <int D>
static hipError_t launch_attn8(const Kv8AttnArgs& a) {
  const Kv8Plan& p = a.p;
  float* const part = static_cast<float*>(a.workspace);
  hipError_t e;
  if (p.max_row >= kKv8TileTokens) {
    float* const tpart = part + chunk_floats(D);
    const int G = p.Hq / p.Hkv;
    const int many = kv8_most_tiles(p.n, p.T, G), few = p.n * kv8_few_tiles(G);
    // 63 single tokens at 4,096 beside a prompt of 512 (D = 256): 73 us, from 512 work-groups 94
    const Kv8Splits splits{tile_pieces((int64_t)many * p.Hkv, D),
                           max(1, (D == 256 ? 384 : 768) / (few * p.Hkv))};
    const dim3 grid(many * splits.many + min(few, p.T) * splits.few + 1, p.Hkv);
    hipLaunchKernelGGL((attn8_tile_kernel<D, kKv8TileWaves>), grid, dim3(64 * kKv8TileWaves), 0,
                       a.stream, a, tpart, splits);
    if (splits.many > 1 || splits.few > 1) {
      if ((e = hipGetLastError()) != hipSuccess) return e;
      const int cut = (splits.many > 1 ? many : 0) + (splits.few > 1 ? few : 0);
      hipLaunchKernelGGL(attn8_join_tiles_kernel<D>, dim3(cut, p.Hkv, kKv8TileWaves),
                         dim3(256), 0,
                         a.stream, a, tpart, splits);
    }
    return hipGetLastError();
  }
  // as many as the rows can have, up to four rounds of the chip's waves
  const int W = kv8_chunk_waves(p.n, p.Hkv);
  const int64_t most = kKv8Waves / W + (int64_t)p.Hkv * min(p.T, p.n * p.max_row);
  const dim3 grid((unsigned)(most < 8192 / W ? most : 8192 / W));
  if (W == 1)
    hipLaunchKernelGGL((attn8_chunk_kernel<D, 1>), grid, dim3(64), 0, a.stream, a, part);
  else
    hipLaunchKernelGGL((attn8_chunk_kernel<D, 4>), grid, dim3(256), 0, a.stream, a, part);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int per = p.max_row;
  const dim3 few(p.n * per, p.Hq);
  hipLaunchKernelGGL(attn8_join_kernel<D>, few, dim3(256), 0, a.stream, a, part, per);
  return hipGetLastError();
}

hipError_t launch_kv8_attn(const Kv8AttnArgs& a) {
  return a.p.D == 256 ? launch_attn8<256>(a) : a.p.D == 128 ? launch_attn8<128>(a) : launch_attn8<64>(a);
}

}  // namespace gdn
