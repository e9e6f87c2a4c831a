// gdn_route.hip -- routing of tokens to experts (SparseMoeBlock's router,
// qwen3_5.rs:226-311): scores, the choice of top_k, and the weights.
//
// One wave per token, lane L holding experts L, L + 64, ... (up to R of them).
// The choice takes the largest score left top_k times. Scores are compared as
// unsigned integers in the floats' order, so that a round is a maximum over the
// lane's R, a DPP maximum over the wave and R equality ballots, the first of
// which that is not empty names the lowest expert with that score.
//   without a bias (and with groups ranked by one score) softmax and sigmoid keep
//     the logits' order: the score is the logit, 32 bits;
//   else it is the score in f64, 64 bits: f32 would make ties of scores that
//     differ. A round then finds the upper halves' maximum and, where several
//     experts have it, the lower halves'.
// Bound by the rounds' VALU work for prompts (16,384 tokens, 256 experts, 8 chosen,
// f32 logits: 11.5 us) and by their latency for decode batches (64 tokens: 4.3 us).
// Where a logit and its expert fit one 32-bit key, moe_route_rows_kernel does four
// tokens a wave.
#include <type_traits>

#include "gdn_common.h"

namespace gdn {
namespace {

// 1 / (1 + exp(-l)), small values with their relative accuracy
__device__ __forceinline__ float sigmoid(float l) {
  const float q = expf(-fabsf(l));
  return (l < 0.f ? q : 1.f) / (1.f + q);
}

// its logarithm, also where it underflows
__device__ __forceinline__ float log_sigmoid(float l) {
  return fminf(l, 0.f) - log1pf(expf(-fabsf(l)));
}

// Largest value of the wave (uniform): four shifts inside the rows of 16 lanes,
// then rows 0 -> 1, 2 -> 3 and 1 -> 2, 3; lane 63 has seen every lane.
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return o > v ? o : v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max_dpp<0x111>(v);  // row_shr:1
  v = max_dpp<0x112>(v);
  v = max_dpp<0x114>(v);
  v = max_dpp<0x118>(v);
  v = max_dpp<0x142>(v);  // row_bcast:15
  v = max_dpp<0x143>(v);  // row_bcast:31
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Floats as unsigned integers in the same order (no NaN; -0 as +0, and both
// above 0, which stands for none).
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ uint64_t ordered(double f) {
  const uint64_t u = (uint64_t)__double_as_longlong(f + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

__device__ __forceinline__ float max_f32(float v) {
  return unordered(wave_max(ordered(v)));
}

// v of lane i (uniform)
__device__ __forceinline__ float of_lane(float v, int i) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
}
__device__ __forceinline__ double of_lane(double v, int i) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), i),
                          __builtin_amdgcn_readlane(__double2loint(v), i));
}

template <int R, bool F64, typename In>
__global__ __launch_bounds__(256) void moe_route_kernel(MoeRouteArgs a) {
  typedef std::conditional_t<F64, double, float> Key;
  extern __shared__ double lds[];  // the wave's scores when there are groups
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * 4 + wave;
  const int E = a.d.num_experts, k = a.d.top_k;
  const int64_t row = (int64_t)min(t, a.T - 1) * a.stride;
  const Key none = -(Key)INFINITY;
  const In* const logits = static_cast<const In*>(a.logits) + row;
  auto clean = [](In raw) {
    float v;
    if constexpr (sizeof(In) == 4)
      v = raw;
    else
      v = bf2f(raw);
    return v != v ? -INFINITY : fminf(v, 3.402823466e38f);
  };
  const bool softmax = a.d.score == GDN_MOE_SOFTMAX;
  In raw[R];  // every load goes out before the first is used
#pragma unroll
  for (int r = 0; r < R; ++r) raw[r] = logits[min(lane + 64 * r, E - 1)];
  const In gate = logits[a.d.shared_gate ? E : 0];
  float bias[F64 ? R : 1];
  if constexpr (F64)
#pragma unroll
    for (int r = 0; r < R; ++r) bias[r] = a.bias ? a.bias[min(lane + 64 * r, E - 1)] : 0.f;
  float l[R];
  float m = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] = lane + 64 * r < E ? clean(raw[r]) : -INFINITY;
    m = fmaxf(m, l[r]);
  }
  // the row's maximum, for softmax's exponentials
  const bool exps = softmax && (F64 || !a.d.renorm);
  if (exps) m = max_f32(m);
  Key key[R];
  if constexpr (F64) {
    // for every expert and without branches, so that the R chains run side by side
    const double top = m > -INFINITY ? (double)m : 0.0;
    double ex[R];
    if (softmax) {
      double sum = 0.0;
#pragma unroll
      for (int r = 0; r < R; ++r) sum += ex[r] = exp((double)l[r] - top);
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
#pragma unroll
      for (int r = 0; r < R; ++r) key[r] = ex[r] / sum;
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) ex[r] = exp(-(double)l[r]);
#pragma unroll
      for (int r = 0; r < R; ++r) key[r] = 1.0 / (1.0 + ex[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (a.bias) key[r] += (double)bias[r];
      key[r] = l[r] > -INFINITY && key[r] == key[r] ? key[r] : none;
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = l[r];
  }
  const int G = a.d.num_groups;
  if (G > 1) {
    Key* const sc = reinterpret_cast<Key*>(lds) + wave * (64 * R);
#pragma unroll
    for (int r = 0; r < R; ++r) sc[lane + 64 * r] = key[r];
    __syncthreads();
    // `per` lanes to a group, so that all of them take part
    int per = 1;
    while (2 * per * G <= 64) per *= 2;
    const int size = E / G, g = lane / per;
    Key b1 = none, b2 = none;  // the group's best two
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
      const Key v = of_lane(gs, o * per);
      before += v > gs || (v == gs && o < g);
    }
    const uint64_t stay = __ballot(before < a.d.top_groups);
    const float inv = 1.0f / (float)size;  // e / size: off by less than the half to spare
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int ge = (int)(((float)(lane + 64 * r) + 0.5f) * inv);
      if (lane + 64 * r < E && !(stay >> (ge * per) & 1)) key[r] = none;
    }
  }
  uint32_t hi[R], lo[F64 ? R : 1];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if constexpr (F64) {
      const uint64_t u = key[r] > none ? ordered(key[r]) : 0;
      hi[r] = (uint32_t)(u >> 32);
      lo[r] = (uint32_t)u;
    } else {
      hi[r] = key[r] > none ? ordered(key[r]) : 0;
    }
  }
  // the choice: lane j keeps the j-th
  int id = -1;
  float lw = -INFINITY;
  for (int j = 0; j < k; ++j) {
    uint32_t best = hi[0];
#pragma unroll
    for (int r = 1; r < R; ++r) best = hi[r] > best ? hi[r] : best;
    const uint32_t M = wave_max(best);
    if (M == 0) break;  // nothing left
    uint32_t L = 0;
    if constexpr (F64) {
      int n = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) n += __popcll(__ballot(hi[r] == M));
      if (n > 1) {
        uint32_t low = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) low = hi[r] == M && lo[r] > low ? lo[r] : low;
        L = wave_max(low);
      }
    }
    float v = 0.f;
    bool open = true;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!open) continue;
      bool eq = hi[r] == M;
      if constexpr (F64) eq = eq && lo[r] >= L;
      const uint64_t b = __ballot(eq);
      if (b == 0) continue;
      open = false;
      const int w = __builtin_ctzll(b);
      if constexpr (F64)
        v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l[r]), w));
      if (lane == w) hi[r] = 0;
      if (lane == j) id = 64 * r + w;
    }
    if constexpr (!F64) v = unordered(M);
    if (lane == j) lw = v;
  }
  // weights, f32; renormalised ones through logarithms, so that scores too small
  // for f32 keep their ratio
  float w;
  if (a.d.renorm) {
    const float base = id < 0 ? -INFINITY : softmax ? lw : log_sigmoid(lw);
    const float bm = max_f32(base);
    const float ex = id < 0 ? 0.f : expf(base - bm);
    w = ex / wave_sum(ex);
  } else if (softmax) {
    float ex = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (l[r] > -INFINITY) ex += expf(l[r] - m);
    w = expf(lw - m) / wave_sum(ex);
  } else {
    w = sigmoid(lw);
  }
  w = id < 0 ? 0.f : w * a.d.scale;
  const int S = a.d.num_shared;
  if (lane >= k && lane < k + S) {
    id = E + lane - k;
    w = a.d.shared_gate ? sigmoid(clean(gate)) : 1.f;
  }
  if (t < a.T && lane < k + S) {
    a.ids[(int64_t)t * (k + S) + lane] = id;
    a.weights[(int64_t)t * (k + S) + lane] = w;
  }
}

// ---- four tokens a wave ----

// Routing on bf16 logits in their own order, without groups, for up to 512 experts
// and 16 columns: 16 lanes (a DPP row) a token, lane L with the R experts from R L on.
// A key is the logit in 16 bits over the expert's number counted down, so that no
// two of a token are equal, the larger one goes first and a tie to the lower
// expert. A round then needs nothing removed: among the keys the next is the one
// with the largest key - last (mod 2^32), since those chosen before, being no
// smaller than the last, come out below all the others. 8 columns of 256 experts:
// 64 tokens 3.2 us (4.3 by a wave a token), 16,384 in 5.2 (11.5), where the logits'
// bytes alone take 1.7; 10 of 512: 3.9 (5.8) and 8.0 (16.6).
typedef short i16x2 __attribute__((ext_vector_type(2)));

// Two logits as 16 bits in order: sign and magnitude to two's complement, turned so
// that the numbers from the lowest finite one to +infinity are 0x0100 .. 0xFFFF and
// -infinity and NaN, which are never chosen, come below; -0 equals +0.
__device__ __forceinline__ uint32_t ordered2(uint32_t v) {
  const i16x2 neg = __builtin_bit_cast(i16x2, v) >> 15;
  const i16x2 mag = __builtin_bit_cast(i16x2, v & 0x7FFF7FFFu);
  const i16x2 base = {(short)0x807F, (short)0x807F};
  return __builtin_bit_cast(uint32_t, (mag ^ neg) - neg + base);
}
constexpr uint32_t kValid = 0x01000000u;  // the lowest key of a number

// The logit of a key, +infinity as the largest float.
__device__ __forceinline__ float key_logit(uint32_t key) {
  const int v = (int)(key >> 16) - 0x807F;
  const float f = __uint_as_float((uint32_t)(v < 0 ? -v : v) << 16);
  return v < 0 ? -f : fminf(f, 3.402823466e38f);
}

// Largest value, or sum, of the row's 16 lanes, in all of them (row_ror:8, 4, 2, 1).
template <int CTRL>
__device__ __forceinline__ uint32_t ror(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, ror<0x128>(v));
  v = max(v, ror<0x124>(v));
  v = max(v, ror<0x122>(v));
  return max(v, ror<0x121>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
  v += __uint_as_float(ror<0x128>(__float_as_uint(v)));
  v += __uint_as_float(ror<0x124>(__float_as_uint(v)));
  v += __uint_as_float(ror<0x122>(__float_as_uint(v)));
  return v + __uint_as_float(ror<0x121>(__float_as_uint(v)));
}

template <int R>
__global__ __launch_bounds__(256) void moe_route_rows_kernel(MoeRouteArgs a) {
  typedef uint32_t Raw __attribute__((ext_vector_type(R / 2), aligned(2)));
  const int L = threadIdx.x & 15, t = blockIdx.x * (blockDim.x >> 4) + (threadIdx.x >> 4);
  const int E = a.d.num_experts, k = a.d.top_k;
  const uint16_t* const logits =
      static_cast<const uint16_t*>(a.logits) + (int64_t)min(t, a.T - 1) * a.stride;
  const uint16_t gate = logits[a.d.shared_gate ? E : 0];
  uint32_t raw[R / 2];
  if (R * (L + 1) <= E) {
    const Raw v = *reinterpret_cast<const Raw*>(logits + R * L);
#pragma unroll
    for (int r = 0; r < R / 2; ++r) raw[r] = v[r];
  } else {  // -infinity past the last expert
#pragma unroll
    for (int r = 0; r < R / 2; ++r) {
      const int e = R * L + 2 * r;
      const uint32_t lo = logits[min(e, E - 1)], hi = logits[min(e + 1, E - 1)];
      raw[r] = (e < E ? lo : 0xFF80u) | (e + 1 < E ? hi : 0xFF80u) << 16;
    }
  }
  uint32_t key[R];
  const uint32_t down = (0xFFFFu - R * L) * 0x10001u - 0x10000u;  // of experts R L and R L + 1
#pragma unroll
  for (int r = 0; r < R / 2; ++r) {
    const uint32_t v = ordered2(raw[r]), e = down - 2 * r * 0x10001u;
    key[2 * r] = v << 16 | (e & 0xFFFFu);
    key[2 * r + 1] = (v & 0xFFFF0000u) | e >> 16;
  }
  // the choice: lane j keeps the j-th key; no number is left once a key is below them
  uint32_t last = 0, mine = 0;
  for (int j = 0; j < k; ++j) {
    uint32_t best = key[0] - last;
#pragma unroll
    for (int r = 1; r < R; ++r) best = max(best, key[r] - last);
    const uint32_t next = last + row16_max(best);
    last = j == 0 || last >= kValid ? next : 0;
    if (L == j) mine = last;
  }
  const bool chosen = mine >= kValid;
  int id = chosen ? (int)(0xFFFFu - (mine & 0xFFFFu)) : -1;
  const bool softmax = a.d.score == GDN_MOE_SOFTMAX;
  const float lw = chosen ? key_logit(mine) : -INFINITY;
  // lane 0 holds the row's largest
  const float top = __shfl(lw, (threadIdx.x & 63) & 48, 64);
  float w;
  if (a.d.renorm) {
    const float ex =
        !chosen ? 0.f : softmax ? expf(lw - top) : expf(log_sigmoid(lw) - log_sigmoid(top));
    w = ex / row16_sum(ex);
  } else if (softmax) {
    float ex = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (key[r] >= kValid) ex += expf(key_logit(key[r]) - top);
    w = expf(lw - top) / row16_sum(ex);
  } else {
    w = sigmoid(lw);
  }
  w = chosen ? w * a.d.scale : 0.f;
  const int S = a.d.num_shared;
  if (L >= k && L < k + S) {
    const float g = bf2f(gate);
    id = E + L - k;
    w = a.d.shared_gate ? sigmoid(g != g ? -INFINITY : fminf(g, 3.402823466e38f)) : 1.f;
  }
  if (t < a.T && L < k + S) {
    a.ids[(int64_t)t * (k + S) + L] = id;
    a.weights[(int64_t)t * (k + S) + L] = w;
  }
}

template <int R>
hipError_t launch_rows(const MoeRouteArgs& a) {
  hipLaunchKernelGGL((moe_route_rows_kernel<R>), dim3((a.T + 15) / 16), dim3(256), 0, a.stream, a);
  return hipGetLastError();
}

template <int R>
hipError_t launch(const MoeRouteArgs& a, bool f64) {
  const size_t bytes = a.d.num_groups > 1 ? 4 * 64 * R * (f64 ? 8 : 4) : 0;
  auto kern = a.d.logits_f32 ? (f64 ? moe_route_kernel<R, true, float> : moe_route_kernel<R, false, float>)
                             : (f64 ? moe_route_kernel<R, true, uint16_t>
                                    : moe_route_kernel<R, false, uint16_t>);
  hipLaunchKernelGGL(kern, dim3((a.T + 3) / 4), dim3(256), bytes, a.stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_route(const MoeRouteArgs& a) {
  const bool f64 = a.bias || (a.d.group_top == 2 && a.d.num_groups > 1);
  const int E = a.d.num_experts;
  if (!f64 && !a.d.logits_f32 && a.d.num_groups == 1 && E <= 512 && a.d.top_k + a.d.num_shared <= 16)
    return E <= 64    ? launch_rows<4>(a)
           : E <= 128 ? launch_rows<8>(a)
           : E <= 256 ? launch_rows<16>(a)
                      : launch_rows<32>(a);
  const int R = (E + 63) / 64;
  return R <= 1   ? launch<1>(a, f64)
         : R <= 2 ? launch<2>(a, f64)
         : R <= 4 ? launch<4>(a, f64)
         : R <= 8 ? launch<8>(a, f64)
                  : launch<16>(a, f64);
}

}  // namespace gdn
