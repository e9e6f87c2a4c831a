// gdn_moe.hip -- the sparse MLP half of a decoder layer: routing of tokens to
// experts and the experts' products on 4-bit weights (SparseMoeBlock,
// qwen3_5.rs:226-311; SwitchMlp, :102-160).
//
// Experts. Entry (t, j) of ids [T, k] names expert e = ids[t, j]:
//   h = silu(Wg_e x_t) * (Wu_e x_t),   out_t = sum_j weights[t, j] * Wd_e h.
// The entries are sorted by expert, the rows of an expert cut into tiles, and
// a work-group takes one tile through some columns of its expert's matrix.
//
// Arithmetic. With groups of 64 k, w = s q + b and X = sum of x over a group, a
// row's product with a column is the sum over the groups of
//   s (sum x (128 + q)) + (b - 128 s) X:
// the nibbles enter the MFMA as the bf16 numbers 128 + q (one v_and_or_b32 per
// two of them), its sums are exact products accumulated in f32, and X comes
// from the same MFMA against ones. h is rounded once to bf16, the operand type
// of its product; out is rounded once from the f32 sum over j.
#include <climits>

#include "gdn_common.h"

namespace gdn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- router --

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}

// 1 / (1 + exp(-l)), small values with their relative accuracy
__device__ __forceinline__ float sigmoid(float l) {
  const float q = expf(-fabsf(l));
  return (l < 0.f ? q : 1.f) / (1.f + q);
}

// its logarithm, also where it underflows
__device__ __forceinline__ float log_sigmoid(float l) {
  return fminf(l, 0.f) - log1pf(expf(-fabsf(l)));
}

// One wave per token, lane L holding experts L R .. L R + R - 1. The score that
// orders the choice is the logit itself (Key = float) or, where a bias or a sum
// of two scores enters, the score in f64: f32 would make ties of scores that
// differ. The best of all lanes' scores is taken top_k times, equal ones by the
// lower index.
template <int R, typename Key>
__global__ __launch_bounds__(256) void moe_route_kernel(MoeRouteArgs a) {
  extern __shared__ double lds[];  // f64 scores per wave when there are groups
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * 4 + wave;
  const int E = a.d.num_experts, k = a.d.top_k;
  const bool here = t < a.T;
  const int64_t row = (int64_t)min(t, a.T - 1) * a.stride;
  const Key none = -(Key)INFINITY;
  constexpr bool kF64 = sizeof(Key) == 8;
  auto logit = [&](int e) {
    float v = a.d.logits_f32 ? static_cast<const float*>(a.logits)[row + e]
                             : bf2f(static_cast<const uint16_t*>(a.logits)[row + e]);
    if (v != v) v = -INFINITY;
    return fminf(v, 3.402823466e38f);
  };
  float l[R];
  float m = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = lane * R + r;
    l[r] = e < E ? logit(e) : -INFINITY;
    m = fmaxf(m, l[r]);
  }
  m = wave_max(m);
  const bool softmax = a.d.score == GDN_MOE_SOFTMAX;
  Key key[R];
  if constexpr (kF64) {
    double sum = 1.0;
    if (softmax && m > -INFINITY) {
      sum = 0.0;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (l[r] > -INFINITY) sum += exp((double)l[r] - (double)m);
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = lane * R + r;
      key[r] = none;
      if (l[r] > -INFINITY) {
        key[r] = softmax ? exp((double)l[r] - (double)m) / sum : 1.0 / (1.0 + exp(-(double)l[r]));
        if (a.bias) key[r] += (double)a.bias[e];
        if (key[r] != key[r]) key[r] = none;
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = l[r];
  }
  const int G = a.d.num_groups;
  if (G > 1) {
    Key* const sc = reinterpret_cast<Key*>(lds) + wave * (64 * R);
#pragma unroll
    for (int r = 0; r < R; ++r) sc[lane * R + r] = key[r];
    __syncthreads();
    // per lanes to a group, so that all of them take part
    int per = 1;
    while (2 * per * G <= 64) per *= 2;
    const int size = E / G, g = lane / per;
    Key b1 = none, b2 = none;
    if (g < G)
      for (int i = lane % per; i < size; i += per) {
        const Key v = sc[g * size + i];
        b2 = v > b1 ? b1 : v > b2 ? v : b2;
        b1 = v > b1 ? v : b1;
      }
    for (int off = 1; off < per; off *= 2) {
      const Key o1 = __shfl_xor(b1, off, 64), o2 = __shfl_xor(b2, off, 64);
      b2 = o1 > b1 ? (b1 > o2 ? b1 : o2) : (o1 > b2 ? o1 : b2);
      b1 = o1 > b1 ? o1 : b1;
    }
    const Key gs = a.d.group_top == 2 && b2 > none ? b1 + b2 : b1;
    // a group stays if fewer than top_groups others go before it
    int before = 0;
    for (int o = 0; o < G; ++o) {
      const Key v = __shfl(gs, o * per, 64);
      before += v > gs || (v == gs && o < g);
    }
    const uint64_t stay = __ballot(before < a.d.top_groups);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = lane * R + r;
      if (e < E && !(stay >> (e / size * per) & 1)) key[r] = none;
    }
  }
  // the choice: lane j keeps the j-th
  int id = -1;
  float lw = -INFINITY;
  for (int j = 0; j < k; ++j) {
    Key best = none;
    float bl = -INFINITY;
    int be = INT_MAX;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (key[r] > best) {
        best = key[r];
        bl = l[r];
        be = lane * R + r;
      }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const Key ob = __shfl_xor(best, off, 64);
      const float ol = __shfl_xor(bl, off, 64);
      const int oe = __shfl_xor(be, off, 64);
      if (ob > best || (ob == best && oe < be)) {
        best = ob;
        bl = ol;
        be = oe;
      }
    }
    if (be == INT_MAX) break;  // nothing left in any lane
    if (lane == j) {
      id = be;
      lw = bl;
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (lane * R + r == be) key[r] = none;
  }
  // weights, f32; renormalised ones through logarithms, so that scores too small
  // for f32 keep their ratio
  float w;
  if (a.d.renorm) {
    const float base = id < 0 ? -INFINITY : softmax ? lw : log_sigmoid(lw);
    const float bm = wave_max(base);
    const float ex = id < 0 ? 0.f : expf(base - bm);
    w = ex / wave_sum(ex);
  } else {
    if (softmax) {
      float ex = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (l[r] > -INFINITY) ex += expf(l[r] - m);
      w = expf(lw - m) / wave_sum(ex);
    } else {
      w = sigmoid(lw);
    }
  }
  w = id < 0 ? 0.f : w * a.d.scale;
  const int S = a.d.num_shared;
  if (lane >= k && lane < k + S) {
    id = E + lane - k;
    w = 1.f;
    if (a.d.shared_gate) {
      const float g = logit(E);
      w = sigmoid(g);
    }
  }
  if (here && lane < k + S) {
    a.ids[(int64_t)t * (k + S) + lane] = id;
    a.weights[(int64_t)t * (k + S) + lane] = w;
  }
}

template <int R>
hipError_t launch_route(const MoeRouteArgs& a, bool by_logit) {
  const size_t lds = a.d.num_groups > 1 ? 4 * 64 * R * (by_logit ? 4 : 8) : 0;
  auto kern = by_logit ? moe_route_kernel<R, float> : moe_route_kernel<R, double>;
  hipLaunchKernelGGL(kern, dim3((a.T + 3) / 4), dim3(256), lds, a.stream, a);
  return hipGetLastError();
}

// --------------------------------------------------------------- packing --

// grid (blocks, experts): expert blockIdx.y's matrix [n, k] into its fragments.
__global__ void moe_pack_kernel(MoePackArgs a) {
  const int P = a.k >> 7, words = a.k >> 3, G = a.k >> 6;
  const int total = (a.n >> 4) * P * 64;
  const int64_t src0 = (int64_t)blockIdx.y * a.n;
  for (int t = blockIdx.x * blockDim.x + threadIdx.x; t < total; t += gridDim.x * blockDim.x) {
    const int lane = t & 63, p = (t >> 6) % P, f = (t >> 6) / P;
    const int r = lane & 15, c = lane >> 4;
    const int64_t n = src0 + 16 * f + r;
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t v = a.w[n * words + 16 * p + 4 * j + c];
      uint32_t q = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q |= ((v >> (8 * i)) & 0xFu) << (4 * i);            // k = 2i     -> nibble i
        q |= ((v >> (8 * i + 4)) & 0xFu) << (4 * (i + 4));  // k = 2i + 1 -> nibble i+4
      }
      o[j] = q;
    }
    const int64_t fp = ((int64_t)blockIdx.y * a.frags + a.fmul * f + a.fofs) * P + p;
    static_cast<u32x4*>(a.wp)[fp * 64 + lane] = o;
    if (lane < 16) {
      const int64_t g = n * G + 2 * p;
      a.sb[fp * 16 + lane] = make_uint2(a.s[g] | (uint32_t)a.s[g + 1] << 16,
                                        a.b[g] | (uint32_t)a.b[g + 1] << 16);
    }
  }
}

// --------------------------------------------------------------- experts --

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// One packed dword -> the operand dwords (128 + q_k0, 128 + q_k1), ... of eight
// consecutive k (m = 0x000F000F held in a VGPR: v_and_or_b32 takes one literal)
__device__ __forceinline__ u32x4 unpack_w(uint32_t w, uint32_t m) {
  const uint32_t e = 0x43004300u;
  return (u32x4){(w & m) | e, ((w >> 4) & m) | e, ((w >> 8) & m) | e, ((w >> 12) & m) | e};
}

// silu(g) * u
__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.0f + expf(-g)) * u; }

constexpr int kTileRows = 16;  // rows of a tile
constexpr int kPassEntries = 1 << 18;

// Work-space of a call: the plan, then the rows between the products.
struct MoeSpace {
  int32_t* ntiles;
  int4* tiles;     // expert, first sorted row, rows, -
  int32_t* perm;   // entry of a sorted row
  uint16_t* h;     // [entries, inner] by sorted row
  float* rows;     // [entries, hidden] by entry
  size_t bytes;
};

int64_t max_tiles(int64_t entries, int experts) {
  return entries / kTileRows + (entries < experts ? entries : experts);
}

MoeSpace moe_space(void* base, int hidden, int inner, int experts, int64_t entries) {
  MoeSpace s{};
  char* const p = static_cast<char*>(base);
  size_t at = 0;
  auto take = [&](size_t n) {
    char* const r = p + at;
    at += (n + 255) & ~(size_t)255;
    return r;
  };
  s.ntiles = reinterpret_cast<int32_t*>(take(4));
  s.tiles = reinterpret_cast<int4*>(take(max_tiles(entries, experts) * sizeof(int4)));
  s.perm = reinterpret_cast<int32_t*>(take(entries * 4));
  s.h = reinterpret_cast<uint16_t*>(take(entries * inner * 2));
  s.rows = reinterpret_cast<float*>(take(entries * hidden * 4));
  s.bytes = at;
  return s;
}

// The plan: a work-group per expert e sorts that expert's entries, in entry
// order, behind those of the experts before it, and lists its tiles. Every
// work-group counts all entries by itself (LDS), so that one launch does it.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void moe_plan_kernel(const int32_t* __restrict__ ids,
                                                                int entries, int experts,
                                                                int32_t* __restrict__ ntiles,
                                                                int4* __restrict__ tiles,
                                                                int32_t* __restrict__ perm) {
  extern __shared__ int cnt[];
  __shared__ int own[kPlanThreads / 64], sums[2][kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = blockIdx.x;
  for (int i = tid; i < experts; i += kPlanThreads) cnt[i] = 0;
  __syncthreads();
  // a wave takes a run of entries, so that its own ones keep their order
  constexpr int W = kPlanThreads / 64;
  const int run = ((entries + W - 1) / W + 63) & ~63;
  const int i0 = wave * run, i1 = min(entries, i0 + run);
  int mine = 0;
  for (int i = i0; i < i1; i += 64) {
    const int id = i + lane < i1 ? ids[i + lane] : -1;
    if ((uint32_t)id < (uint32_t)experts) atomicAdd(&cnt[id], 1);
    mine += __popcll(__ballot(id == e));
  }
  if (lane == 0) own[wave] = mine;
  __syncthreads();
  int before = 0, tbefore = 0;
  for (int i = tid; i < experts; i += kPlanThreads) {
    const int c = cnt[i], n = (c + kTileRows - 1) / kTileRows;
    before += i < e ? c : 0;
    tbefore += i < e ? n : 0;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    before += __shfl_xor(before, off, 64);
    tbefore += __shfl_xor(tbefore, off, 64);
  }
  if (lane == 0) {
    sums[0][wave] = before;
    sums[1][wave] = tbefore;
  }
  __syncthreads();
  before = tbefore = 0;
  int at = 0;
  for (int w = 0; w < W; ++w) {
    before += sums[0][w];
    tbefore += sums[1][w];
    if (w < wave) at += own[w];
  }
  const int n = cnt[e], nt = (n + kTileRows - 1) / kTileRows;
  if (e == experts - 1 && tid == 0) *ntiles = tbefore + nt;
  for (int i = tid; i < nt; i += kPlanThreads)
    tiles[tbefore + i] = make_int4(e, before + kTileRows * i, min(kTileRows, n - kTileRows * i), 0);
  if (mine == 0) return;
  at += before;
  for (int i = i0; i < i1; i += 64) {
    const bool hit = i + lane < i1 && ids[i + lane] == e;
    const uint64_t b = __ballot(hit);
    if (hit) perm[at + __popcll(b & ((1ull << lane) - 1))] = i + lane;
    at += __popcll(b);
  }
}

// One 16-row tile against NF 16-column fragments over the stages p0, p0 + 1,
// ..., 4 at a time: every load of the four goes out before the first product.
// x is the MFMA A operand, so lane (r16, c4) supplies row r16 (zeros past the
// tile's rows) and ends with rows 4 c4 + i, column r16 of each fragment: one
// scale and one offset per group for all of its sums.
template <int NF>
__device__ __forceinline__ void tile_product(const uint16_t* xrow, bool live,
                                             const u32x4* wp, const uint2* sb, int P, int p0,
                                             int step, f32x4 (&T)[NF]) {
  const int lane = threadIdx.x & 63, r16 = lane & 15, c4 = lane >> 4;
  const u32x4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  uint32_t nib = 0x000F000Fu;
  asm volatile("" : "+v"(nib));
#pragma unroll
  for (int f = 0; f < NF; ++f) T[f] = zero;
  for (; p0 < P; p0 += step) {
    u32x4 w[4][NF], X[4][4];
    uint2 s[4][NF];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int p = min(p0 + q, P - 1);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        w[q][f] = __builtin_nontemporal_load(wp + ((int64_t)f * P + p) * 64 + lane);
        s[q][f] = sb[((int64_t)f * P + p) * 16 + r16];
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int p = min(p0 + q, P - 1);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        X[q][h] = (u32x4){0u, 0u, 0u, 0u};
        if (live) X[q][h] = *reinterpret_cast<const u32x4*>(xrow + 128 * p + 32 * h + 8 * c4);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (p0 + q >= P) break;
#pragma unroll
      for (int gl = 0; gl < 2; ++gl) {
        f32x4 xg = mfma(X[q][2 * gl], ones, zero);
        xg = mfma(X[q][2 * gl + 1], ones, xg);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          f32x4 d = mfma(X[q][2 * gl], unpack_w(w[q][f][2 * gl], nib), zero);
          d = mfma(X[q][2 * gl + 1], unpack_w(w[q][f][2 * gl + 1], nib), d);
          const float sc = gl ? bf_hi(s[q][f].x) : bf_lo(s[q][f].x);
          const float of = fmaf(-128.0f, sc, gl ? bf_hi(s[q][f].y) : bf_lo(s[q][f].y));
#pragma unroll
          for (int i = 0; i < 4; ++i) T[f][i] = fmaf(sc, d[i], fmaf(of, xg[i], T[f][i]));
        }
      }
    }
  }
}

// h of one tile's rows, 16 inner columns: work-group (tile, column block) of
// four waves, each over a quarter of the stages, added in wave order.
__global__ __launch_bounds__(256) void moe_up_kernel(MoeArgs a, MoeSpace s) {
  const int blocks = a.inner / 16;
  const int tile = blockIdx.x / blocks, j = blockIdx.x - tile * blocks;
  if (tile >= *s.ntiles) return;
  __shared__ f32x4 part[4][2][64];
  const int4 tl = s.tiles[tile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15;
  const int P = a.hidden >> 7;
  const int row = min(r16, tl.z - 1);
  const uint16_t* const xrow = a.x + (int64_t)(s.perm[tl.y + row] / a.k) * a.xs;
  const int64_t f = ((int64_t)tl.x * blocks + j) * 2 * P;
  f32x4 T[2];
  tile_product<2>(xrow, r16 < tl.z, static_cast<const u32x4*>(a.w1) + f * 64, a.sb1 + f * 16, P,
                  4 * wave, 16, T);
  part[wave][0][lane] = T[0];
  part[wave][1][lane] = T[1];
  __syncthreads();
  // thread (element i of lane l): row 4 (l / 16) + i, column l % 16
  const int l = threadIdx.x >> 2, i = threadIdx.x & 3, m = 4 * (l >> 4) + i;
  float g = 0.f, u = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    g += part[w][0][l][i];
    u += part[w][1][l][i];
  }
  if (m < tl.z) s.h[(int64_t)(tl.y + m) * a.inner + 16 * j + (l & 15)] = f2bf(swiglu(g, u));
}

// The weighted rows of down: a wave per 32 columns of a tile.
__global__ __launch_bounds__(256) void moe_down_kernel(MoeArgs a, MoeSpace s) {
  const int blocks = a.hidden / 128;
  const int tile = blockIdx.x / blocks, cb = blockIdx.x - tile * blocks;
  if (tile >= *s.ntiles) return;
  const int4 tl = s.tiles[tile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, c4 = lane >> 4;
  const int P = a.inner >> 7, f0 = cb * 8 + 2 * wave;
  const uint16_t* const hrow = s.h + (int64_t)(tl.y + min(r16, tl.z - 1)) * a.inner;
  const int64_t f = ((int64_t)tl.x * (a.hidden / 16) + f0) * P;
  f32x4 T[2];
  tile_product<2>(hrow, r16 < tl.z, static_cast<const u32x4*>(a.w2) + f * 64, a.sb2 + f * 16, P, 0,
                  4, T);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = 4 * c4 + i;
    if (m >= tl.z) continue;
    const int en = s.perm[tl.y + m];
    const float wt = a.weights[en];
    float* const o = s.rows + (int64_t)en * a.hidden + 16 * f0 + r16;
    o[0] = wt * T[0][i];
    o[16] = wt * T[1][i];
  }
}

// out[t] = the sum of its entries' rows in column order. A thread per 4 columns.
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs a, MoeSpace s) {
  const int q = a.hidden / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.T * q) return;
  const int64_t t = i / q;
  const int c = (int)(i - t * q) * 4;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.k; ++j)
    if ((uint32_t)a.ids[t * a.k + j] < (uint32_t)a.experts)
      y += *reinterpret_cast<const f32x4*>(s.rows + (t * a.k + j) * a.hidden + c);
  *reinterpret_cast<u32x2*>(a.out + t * a.os + c) = (u32x2){f2bf2(y[0], y[1]), f2bf2(y[2], y[3])};
}

}  // namespace

hipError_t launch_moe_route(const MoeRouteArgs& a) {
  const bool by_logit = !a.bias && (a.d.group_top == 1 || a.d.num_groups == 1);
  const int R = (a.d.num_experts + 63) / 64;
  return R <= 1   ? launch_route<1>(a, by_logit)
         : R <= 2 ? launch_route<2>(a, by_logit)
         : R <= 4 ? launch_route<4>(a, by_logit)
         : R <= 8 ? launch_route<8>(a, by_logit)
                  : launch_route<16>(a, by_logit);
}

hipError_t launch_moe_pack(const MoePackArgs& a) {
  const int blocks = (a.n * (a.k / 128) * 4 + 255) / 256;
  hipLaunchKernelGGL(moe_pack_kernel, dim3(blocks < 64 ? blocks : 64, a.experts), dim3(256), 0,
                     a.stream, a);
  return hipGetLastError();
}

int moe_pass_tokens(int k, int64_t x_stride) {
  (void)x_stride;
  return kPassEntries / k;
}

size_t moe_workspace_bytes(int hidden, int inner, int experts, int T, int k) {
  const int64_t entries = (int64_t)T * k;
  return moe_space(nullptr, hidden, inner, experts, entries < kPassEntries ? entries : kPassEntries)
      .bytes;
}

hipError_t launch_moe(const MoeArgs& a) {
  const int entries = a.T * a.k;
  const MoeSpace s = moe_space(a.workspace, a.hidden, a.inner, a.experts, entries);
  const unsigned tiles = (unsigned)max_tiles(entries, a.experts);
  hipLaunchKernelGGL(moe_plan_kernel, dim3(a.experts), dim3(kPlanThreads), a.experts * 4, a.stream,
                     a.ids, entries, a.experts, s.ntiles, s.tiles, s.perm);
  hipLaunchKernelGGL(moe_up_kernel, dim3(tiles * (a.inner / 16)), dim3(256), 0, a.stream, a, s);
  hipLaunchKernelGGL(moe_down_kernel, dim3(tiles * (a.hidden / 128)), dim3(256), 0, a.stream, a, s);
  const int64_t n = (int64_t)a.T * (a.hidden / 4);
  hipLaunchKernelGGL(moe_combine_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, a.stream,
                     a, s);
  return hipGetLastError();
}

}  // namespace gdn
