// gdn_norm.hip -- the norms behind and before a block in one pass over its rows:
//   b  = x * rsqrt(mean(x^2) + eps) * post_w            (or x)
//   h' = h + scale * gate * b
//   hn = h' * rsqrt(mean(h'^2) + eps') * pre_w
// Both means are sums over a row, so a work-group holds one row in registers
// (f32) from its only read to its only write. h' enters the second norm before
// its rounding to the residual stream's type.
// Bound by HBM: 16,384 rows of 2048 in bf16 take 40 us, 268 MB at 6.6 TB/s; 64 rows by
// the latency of a launch, the loads and two sums, 3.5 us.
#include "gdn_common.h"

namespace gdn {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void unpack8(u32x4 v, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf_lo(v[i]);
    f[2 * i + 1] = bf_hi(v[i]);
  }
}

__device__ __forceinline__ u32x4 pack8(const float* f) {
  return (u32x4){f2bf2(f[0], f[1]), f2bf2(f[2], f[3]), f2bf2(f[4], f[5]), f2bf2(f[6], f[7])};
}

// Sum over the work-group's threads, the same bits in all of them; red holds
// one float per wave.
template <int TH>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (TH > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TH / 64; ++i) v += red[i];
  }
  return v;
}

// One row per group of TH threads; thread t holds the 8 elements from
// 8 t + 8 TH j, j < J. grid n, block TH.
template <int TH, int J, bool F32>
__global__ __launch_bounds__(TH) void block_norm_kernel(BlockNormArgs a) {
  __shared__ float red[2][TH / 64];
  const int hidden = a.d.hidden, tid = threadIdx.x;
  const int64_t i = blockIdx.x;
  const uint16_t* const xr = a.x + i * a.x_stride;
  u32x4 xv[J], hv[J][F32 ? 2 : 1], pw[J], qw[J], gv[J];
  const bool elem = a.d.gate == GDN_GATE_ELEMENT;
  // every load of the row goes out before the first sum
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = 8 * (tid + TH * j);
    if (c < hidden) {
      xv[j] = *reinterpret_cast<const u32x4*>(xr + c);
      if constexpr (F32) {
        const float* const hr = static_cast<const float*>(a.h) + i * a.h_stride;
        hv[j][0] = *reinterpret_cast<const u32x4*>(hr + c);
        hv[j][1] = *reinterpret_cast<const u32x4*>(hr + c + 4);
      } else {
        const uint16_t* const hr = static_cast<const uint16_t*>(a.h) + i * a.h_stride;
        hv[j][0] = *reinterpret_cast<const u32x4*>(hr + c);
      }
      if (elem) gv[j] = *reinterpret_cast<const u32x4*>(a.gate + i * a.gate_stride + c);
      if (a.post_w) pw[j] = *reinterpret_cast<const u32x4*>(a.post_w + c);
      if (a.pre_w) qw[j] = *reinterpret_cast<const u32x4*>(a.pre_w + c);
    }
  }
  float scale = a.d.scale;
  if (a.d.gate == GDN_GATE_ROW) {
    const float g = bf2f(a.gate[i * a.gate_stride]);
    scale *= a.d.gate_sigmoid ? 1.0f / (1.0f + expf(-g)) : g;
  }
  const float one = a.d.unit_offset ? 1.0f : 0.0f;
  if (a.post_w) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (8 * (tid + TH * j) < hidden) {
        float f[8];
        unpack8(xv[j], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
      }
    scale *= 1.0f / sqrtf(row_sum<TH>(ss, red[0]) / (float)hidden + a.d.post_eps);
  }
  float y[J][8];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = 8 * (tid + TH * j);
    if (c < hidden) {
      float f[8], g[8];
      unpack8(xv[j], f);
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[j][e] = __uint_as_float(hv[j][e >> 2][e & 3]);
      } else {
        unpack8(hv[j][0], y[j]);
      }
      if (elem) {
        unpack8(gv[j], g);
        if (a.d.gate_sigmoid)
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = 1.0f / (1.0f + expf(-g[e]));
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= g[e];
      }
      if (a.post_w) {
        unpack8(pw[j], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= one + g[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[j][e] = fmaf(scale, f[e], y[j][e]);
        ss = fmaf(y[j][e], y[j][e], ss);
      }
      if constexpr (F32) {
        float* const o = static_cast<float*>(a.h_out) + i * a.h_out_stride + c;
        *reinterpret_cast<v4f*>(o) = (v4f){y[j][0], y[j][1], y[j][2], y[j][3]};
        *reinterpret_cast<v4f*>(o + 4) = (v4f){y[j][4], y[j][5], y[j][6], y[j][7]};
      } else {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.h_out) + i * a.h_out_stride + c) =
            pack8(y[j]);
      }
    }
  }
  if (!a.pre_w) return;
  const float r = 1.0f / sqrtf(row_sum<TH>(ss, red[1]) / (float)hidden + a.d.pre_eps);
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int c = 8 * (tid + TH * j);
    if (c < hidden) {
      float g[8];
      unpack8(qw[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[j][e] *= r * (one + g[e]);
      *reinterpret_cast<u32x4*>(a.hn + i * a.hn_stride + c) = pack8(y[j]);
    }
  }
}

template <int TH, int J>
hipError_t launch(const BlockNormArgs& a) {
  auto kern = a.d.h_f32 ? block_norm_kernel<TH, J, true> : block_norm_kernel<TH, J, false>;
  hipLaunchKernelGGL(kern, dim3(a.n), dim3(TH), 0, a.stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_norm(const BlockNormArgs& a) {
  const int h = a.d.hidden;
  if (h <= 512) return launch<64, 1>(a);
  if (h <= 2048) return launch<256, 1>(a);
  if (h <= 4096) return launch<256, 2>(a);
  if (h <= 8192) return launch<256, 4>(a);
  return launch<512, 4>(a);
}

}  // namespace gdn
