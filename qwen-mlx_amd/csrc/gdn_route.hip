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
// Bound by the rounds' VALU work for prompts (16,384 tokens, 256 experts, 8 chosen:
// 12.7 us) and by their latency for decode batches (64 tokens: 4.6 us).
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
      key[r] = none;
      if (l[r] > -INFINITY) {
        key[r] = softmax ? exp((double)l[r] - (double)m) / sum : 1.0 / (1.0 + exp(-(double)l[r]));
        if (a.bias) key[r] += (double)a.bias[lane + 64 * r];
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
      const Key v = __shfl(gs, o * per, 64);
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
  const int R = (a.d.num_experts + 63) / 64;
  return R <= 1   ? launch<1>(a, f64)
         : R <= 2 ? launch<2>(a, f64)
         : R <= 4 ? launch<4>(a, f64)
         : R <= 8 ? launch<8>(a, f64)
                  : launch<16>(a, f64);
}

}  // namespace gdn
