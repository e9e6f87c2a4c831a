// gdn_rope.hip -- rotary positions of q and k heads, with their norms:
//   y = x * w / sqrt(mean(x^2) + eps)   (or x)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_a sin + y_b cos) of pair i at pos * f_i
// The angle in turns is a product in 64 bits, of which the fraction goes on in f32: at
// position 10^6 an f32 product would be off by 2^-5 turns.
// Bound by HBM: each element is read and written once; 16,384 tokens of 18 bf16 heads of 256 dims,
// 302 MB, 59 us (5.1 TB/s where a large copy reaches 5.2), 64 of them 4 us.
#include "gdn_common.h"

namespace gdn {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 8 elements of a head as loaded: 4 words of bf16, or 8 of f32
template <bool F32>
struct Raw {
  u32x4 v[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    const u32x4* s = F32 ? reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + i)
                         : reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int k = 0; k < (F32 ? 2 : 1); ++k) v[k] = __builtin_nontemporal_load(s + k);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < (F32 ? 2 : 1); ++k) v[k] = (u32x4){0u, 0u, 0u, 0u};
  }
  __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      f[k] = F32 ? __uint_as_float(v[F32 ? k >> 2 : 0][k & 3])
                 : k & 1 ? bf_hi(v[0][k >> 1]) : bf_lo(v[0][k >> 1]);
  }
  // the same elements of another lane
  __device__ __forceinline__ Raw from(int lane) const {
    Raw r;
#pragma unroll
    for (int k = 0; k < (F32 ? 2 : 1); ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) r.v[k][w] = __shfl(v[k][w], lane, 64);
    return r;
  }
};

template <bool F32>
__device__ __forceinline__ void store8(void* p, int64_t i, const float* f) {
  if constexpr (F32) {
    v4f* d = reinterpret_cast<v4f*>(static_cast<float*>(p) + i);
    __builtin_nontemporal_store((v4f){f[0], f[1], f[2], f[3]}, d);
    __builtin_nontemporal_store((v4f){f[4], f[5], f[6], f[7]}, d + 1);
  } else {
    __builtin_nontemporal_store(
        (u32x4){f2bf2(f[0], f[1]), f2bf2(f[2], f[3]), f2bf2(f[4], f[5]), f2bf2(f[6], f[7])},
        reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i));
  }
}

// Sum over the LH lanes of a head (aligned), the same bits in all of them.
template <int LH>
__device__ __forceinline__ float head_sum(float v) {
  if constexpr (LH >= 2) v += dpp_quad_xor1(v);
  if constexpr (LH >= 4) v += dpp_quad_xor2(v);
  if constexpr (LH >= 8) v += dpp_half_mirror(v);
  if constexpr (LH >= 16)
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, false));
  if constexpr (LH >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (LH >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Pairs: neighbours in a lane; elements of two lanes (rotary_dim a multiple of 16), whose
// elements come by a lane exchange before the norm; or anywhere, through LDS after it.
enum { kNeighbours, kLanes, kAnywhere };

// Work-group of four waves: `tokens` tokens, WPT waves a token, a head in LH lanes of 8 dims. The
// work-group forms its tokens' sines and cosines in LDS first, a pair a thread at a time;
// a wave then goes through its token's heads (grid y: a part of them), kAhead loads in flight.
template <bool F32, int LH, int PAIRS>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int tokens, int wpt) {
  constexpr int kHeads = 64 / LH;  // of a wave at once
  constexpr int kAhead = 3;
  extern __shared__ float lds[];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane % LH;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = a.rot >> 1, t0 = blockIdx.x * tokens;
  const int nt = min(tokens, a.T - t0);
  float* const cs = lds;
  float* const sn = cs + tokens * half;
  float* const xs = sn + tokens * half + wave * 512;  // kAnywhere: 64 lanes' elements
  for (int i = tid; i < nt * half; i += 256) {
    const int k = i / half;
    double turns = (double)a.pos[t0 + k] * a.turns[i - k * half];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[i] = c * a.mag;
    sn[i] = (a.inverse ? -s : s) * a.mag;
  }
  __syncthreads();
  const int d0 = 8 * hl;
  const bool in = d0 < a.D;
  const int lanes = half >> 3;  // kLanes: lanes of a half
  const bool second = d0 >= half;
  const int other = lane + (PAIRS == kLanes && d0 < a.rot ? (second ? -lanes : lanes) : 0);
  const int od = PAIRS == kLanes && d0 < a.rot ? (second ? d0 - half : d0 + half) : d0;
  // q's heads, then k's, kHeads at a time; one part of them for each grid y and each of a
  // token's waves
  const int qg = (a.q.heads + kHeads - 1) / kHeads, groups = qg + (a.k.heads + kHeads - 1) / kHeads;
  const int parts = gridDim.y * wpt, gpp = (groups + parts - 1) / parts;
  const int g0 = (blockIdx.y * wpt + wave % wpt) * gpp, g1 = min(g0 + gpp, groups);
  const float inv_dim = 1.0f / (float)a.D;
  for (int k = wave / wpt; k < nt; k += 4 / wpt) {
    const int64_t t = t0 + k;
    const bool stay = a.pos[t] < 0;
    bool turned[8];
    float c[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      const int i = PAIRS == kNeighbours ? d >> 1 : d < half ? d : d - half;
      // lanes' pairs: all of a lane's or none
      turned[e] = (PAIRS == kLanes ? d0 : d) < a.rot && !stay;
      c[e] = turned[e] ? cs[k * half + i] : 1.f;
      s[e] = turned[e] ? sn[k * half + i] : 0.f;
      if (PAIRS == kNeighbours ? !(d & 1) : d < half) s[e] = -s[e];
    }
    auto head = [&](int g) __attribute__((always_inline)) {
      return (g < qg ? g : g - qg) * kHeads + lane / LH;
    };
    Raw<F32> x[kAhead];
    auto load = [&](int g, Raw<F32>& r) __attribute__((always_inline)) {
      const gdn_rope_rows& w = g < qg ? a.q : a.k;
      const int j = head(g);
      r.zero();
      if (j < w.heads && in) r.load(w.in, t * w.in_stride + j * w.in_head_stride + d0);
    };
    float wy[8], wo[8];  // norm weights of the lane's elements and of their partners
    int have = -1;       // of q (1) or k (0)
    auto turn = [&](int g, const Raw<F32>& r) __attribute__((always_inline)) {
      const bool isq = g < qg;
      const gdn_rope_rows& w = isq ? a.q : a.k;
      const int j = head(g);
      float y[8], o[8];
      r.floats(y);
      if constexpr (PAIRS == kLanes) r.from(other).floats(o);
      if (w.norm_w && !stay) {
        if (have != (int)isq) {
          have = (int)isq;
          Raw<false> r0, r1;
          r0.zero();
          r1.zero();
          if (in) {
            r0.load(w.norm_w, d0);
            if (PAIRS == kLanes) r1.load(w.norm_w, od);
          }
          r0.floats(wy);
          r1.floats(wo);
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
        const float rn = 1.0f / sqrtf(fmaf(head_sum<LH>(ss), inv_dim, a.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] *= rn * wy[e];
          if constexpr (PAIRS == kLanes) o[e] *= rn * wo[e];
        }
      }
      if constexpr (PAIRS == kNeighbours) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = y[e ^ 1];
      }
      if constexpr (PAIRS == kAnywhere) {
#pragma unroll
        for (int e = 0; e < 8; ++e) xs[8 * lane + e] = y[e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = d0 + e;
          o[e] = xs[8 * (lane - hl) + (d >= a.rot ? d : d < half ? d + half : d - half)];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
      }
      // what does not turn does not meet its partner, which may be anything
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = turned[e] ? fmaf(o[e], s[e], y[e] * c[e]) : y[e];
      if (j < w.heads && in) store8<F32>(w.out, t * w.out_stride + j * w.out_head_stride + d0, y);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (g0 + i < g1) load(g0 + i, x[i]);
    for (int g = g0; g < g1; g += kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (g + i >= g1) break;
        turn(g + i, x[i]);
        if (g + i + kAhead < g1) load(g + i + kAhead, x[i]);
      }
    }
  }
}

template <bool F32, int LH>
hipError_t launch_pairs(const RopeArgs& a) {
  const int groups = (a.q.heads + 64 / LH - 1) / (64 / LH) + (a.k.heads + 64 / LH - 1) / (64 / LH);
  // long steps: two tokens a wave; short ones: a token's heads over the waves of several
  // work-groups, one round each. 18 heads of 256 dims, short / long: 512 tokens 9 / 16 us, 1,024
  // 13 / 18, 2,048 21 / 19, 4,096 38 / 23.
  const bool many = a.T >= 2048;
  const int tokens = many ? 8 : 1, wpt = many ? 1 : 4;
  const dim3 grid((a.T + tokens - 1) / tokens, many ? 1 : (groups + wpt - 1) / wpt);
  size_t bytes = (size_t)tokens * a.rot * sizeof(float);
  if (a.interleaved) {
    hipLaunchKernelGGL((rope_kernel<F32, LH, kNeighbours>), grid, dim3(256), bytes, a.stream, a, tokens, wpt);
  } else if (a.rot % 16 == 0) {
    hipLaunchKernelGGL((rope_kernel<F32, LH, kLanes>), grid, dim3(256), bytes, a.stream, a, tokens, wpt);
  } else {
    bytes += 4 * 512 * sizeof(float);
    hipLaunchKernelGGL((rope_kernel<F32, LH, kAnywhere>), grid, dim3(256), bytes, a.stream, a, tokens, wpt);
  }
  return hipGetLastError();
}

template <bool F32>
hipError_t launch_lanes(const RopeArgs& a) {
  const int lanes = a.D / 8;
  return lanes <= 8    ? launch_pairs<F32, 8>(a)
         : lanes <= 16 ? launch_pairs<F32, 16>(a)
         : lanes <= 32 ? launch_pairs<F32, 32>(a)
                       : launch_pairs<F32, 64>(a);
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a) {
  return a.f32 ? launch_lanes<true>(a) : launch_lanes<false>(a);
}

}  // namespace gdn
