// gdn_rope.hip -- rotary positions of q and k heads, with their norms:
//   y = x * w / sqrt(mean(x^2) + eps)   (or x)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_a sin + y_b cos) of pair i at pos * f_i
// The angle in turns is a product in 64 bits, of which the fraction goes on in f32: at
// position 10^6 an f32 product would be off by 2^-5 turns.
// Bound by HBM: each element is read and written once.
#include "gdn_common.h"

namespace gdn {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <bool F32>
__device__ __forceinline__ void load8(const void* p, int64_t i, float* f) {
  if constexpr (F32) {
    const v4f* s = reinterpret_cast<const v4f*>(static_cast<const float*>(p) + i);
    const v4f a = s[0], b = s[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[k] = a[k];
      f[4 + k] = b[k];
    }
  } else {
    const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = bf_lo(v[k]);
      f[2 * k + 1] = bf_hi(v[k]);
    }
  }
}

template <bool F32>
__device__ __forceinline__ void store8(void* p, int64_t i, const float* f) {
  if constexpr (F32) {
    v4f* d = reinterpret_cast<v4f*>(static_cast<float*>(p) + i);
    d[0] = (v4f){f[0], f[1], f[2], f[3]};
    d[1] = (v4f){f[4], f[5], f[6], f[7]};
  } else {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) =
        (u32x4){f2bf2(f[0], f[1]), f2bf2(f[2], f[3]), f2bf2(f[4], f[5]), f2bf2(f[6], f[7])};
  }
}

// Work-group: a token and up to hpg of its heads, a wave a head at a time with the head in
// LDS, 8 dims a lane. block 256.
template <bool F32>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int hpg) {
  __shared__ float cs[256], sn[256];
  __shared__ float xs[4][512];
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pos = a.pos[t];
  const int rot = pos < 0 ? 0 : a.rot, half = rot >> 1;
  for (int i = tid; i < half; i += 256) {
    double turns = (double)pos * a.turns[i];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[i] = c * a.mag;
    sn[i] = (a.inverse ? -s : s) * a.mag;
  }
  __syncthreads();
  const int heads = a.q.heads + a.k.heads;
  const int h1 = min((int)(blockIdx.y + 1) * hpg, heads);
  const int d0 = 8 * lane;
  for (int h = blockIdx.y * hpg + wave; h < h1; h += 4) {
    const bool isq = h < a.q.heads;
    const gdn_rope_rows& r = isq ? a.q : a.k;
    const int j = isq ? h : h - a.q.heads;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (d0 < a.D) load8<F32>(r.in, t * r.in_stride + j * r.in_head_stride + d0, x);
    if (r.norm_w && pos >= 0) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
      const float rn = 1.0f / sqrtf(wave_sum(ss) / (float)a.D + a.eps);
      float w[8];
      if (d0 < a.D) load8<false>(r.norm_w, d0, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = x[k] * rn * w[k];
    }
    if (d0 < a.D) {
#pragma unroll
      for (int k = 0; k < 8; ++k) xs[wave][d0 + k] = x[k];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    if (d0 < a.D) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int d = d0 + k;
        if (d >= rot) continue;
        const int i = a.interleaved ? d >> 1 : d < half ? d : d - half;
        const bool second = a.interleaved ? (d & 1) : d >= half;
        const float o = xs[wave][a.interleaved ? d ^ 1 : second ? d - half : d + half];
        x[k] = second ? o * sn[i] + x[k] * cs[i] : x[k] * cs[i] - o * sn[i];
      }
      store8<F32>(r.out, t * r.out_stride + j * r.out_head_stride + d0, x);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a) {
  const int heads = a.q.heads + a.k.heads;
  const int hpg = a.T >= 512 ? heads : 4;
  const dim3 grid(a.T, (heads + hpg - 1) / hpg);
  if (a.f32)
    hipLaunchKernelGGL(rope_kernel<true>, grid, dim3(256), 0, a.stream, a, hpg);
  else
    hipLaunchKernelGGL(rope_kernel<false>, grid, dim3(256), 0, a.stream, a, hpg);
  return hipGetLastError();
}

}  // namespace gdn
