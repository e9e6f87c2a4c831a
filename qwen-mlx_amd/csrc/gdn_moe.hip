// gdn_moe.hip -- the experts' products on 4-bit weights (SwitchMlp,
// qwen3_5.rs:102-160; SharedExpert, :164-222).
//
// Entry (t, j) of ids [T, k] names expert e = ids[t, j]:
//   h = silu(Wg_e x_t) * (Wu_e x_t),   out_t = sum_j weights[t, j] * Wd_e h.
// The entries are sorted by expert, the rows of an expert cut into tiles, and
// a work-group takes one tile through some columns of its expert's matrix.
//
// Arithmetic. With groups of 64 k, w = s q + b and X = sum of x over a group, a
// row's product with a column is the sum over the groups of
//   s (sum x (128 + q)) + (b - 128 s) X:
// the nibbles enter the MFMA as the bf16 numbers 128 + q (one v_and_or_b32 per
// two of them), its sums are exact products accumulated in f32, and X comes
// from the same MFMA against ones.
// h enters down's product, at the same rate, as f16 times a power of two of its row
// (11 bits; as bf16 the result's error was 0.0025 of its norm, 0.0017 of which is its
// own rounding), and the nibbles as the f16 numbers 1024 + q. The power is known
// before h is: with S_g and S_u the largest sums of |w| over a row of the expert's
// gate and up, |h| <= |g| |u| <= S_g S_u max|x|^2, and this is brought to 2^15 at
// most (row_exponent). A value has its 11 bits down to 2^-29 of that. Calls of very
// few entries have h in two bf16 parts instead. out is rounded once from the f32 sum
// over j, whose rows are f32 or, of long prompts, f16 under an exponent per row
// (moe_wide_down_kernel).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "gdn_common.h"

namespace gdn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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
    if (lane < 32) {  // lanes 0-15 the scales of rows r, 16-31 their biases
      const uint16_t* const v = lane < 16 ? a.s : a.b;
      const int64_t g = n * G + 2 * p;
      a.sb[fp * 32 + lane] = v[g] | (uint32_t)v[g + 1] << 16;
    }
  }
}

// bound[e] = the largest sum of |w| over a row of expert e's matrix [n, k] whose sum is
// finite; bound starts at zeros. Every term counts 2^-16 of the magnitudes that its
// products with the numbers offset + q pass through as well: weights that cancel to
// less than the f32 sums' error leave that. grid (n / 64 rounded up, experts), a wave
// 16 rows, four lanes a row. Positive floats are in the order of their bits, and a
// maximum has no order.
__global__ __launch_bounds__(256) void moe_bound_kernel(MoePackArgs a, float offset, float* bound) {
  const int lane = threadIdx.x & 63, c = lane & 3;
  const int n = blockIdx.x * 64 + (threadIdx.x >> 6) * 16 + (lane >> 2);
  const int words = a.k >> 3, G = a.k >> 6;
  float sum = 0.f;
  if (n < a.n) {
    const int64_t row = (int64_t)blockIdx.y * a.n + n;
    for (int j = 4 * c; j < words; j += 16) {
      const float sc = bf2f(a.s[row * G + (j >> 3)]), of = bf2f(a.b[row * G + (j >> 3)]);
      const float err = 0x1p-16f * fmaf(2.0f * offset + 15.0f, fabsf(sc), fabsf(of));
      sum = fmaf(32.0f, err, sum);  // the lane's 32 terms
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t v = a.w[row * words + j + q];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += fabsf(fmaf(sc, (float)(v >> (4 * i) & 15), of));
      }
    }
  }
  sum += __shfl_xor(sum, 1, 64);
  sum += __shfl_xor(sum, 2, 64);
  if (!(sum < INFINITY)) sum = 0.f;
#pragma unroll
  for (int off = 4; off < 64; off *= 2) sum = fmaxf(sum, __shfl_xor(sum, off, 64));
  if (lane == 0) atomicMax(reinterpret_cast<int*>(bound) + blockIdx.y, __float_as_int(sum));
}

// --------------------------------------------------------------- experts --

// The products' operands: bf16, or f16 for H (rows of h).
template <bool H = false>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (H)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// What a nibble's number is above it: the type's first power of two with steps of one.
constexpr float kOffsetX = 128.0f, kOffsetH = 1024.0f;

// One packed dword -> the operand dwords (offset + q_k0, offset + q_k1), ... of eight
// consecutive k (m = 0x000F000F held in a VGPR: v_and_or_b32 takes one literal)
template <bool H = false>
__device__ __forceinline__ u32x4 unpack_w(uint32_t w, uint32_t m) {
  const uint32_t e = H ? 0x64006400u : 0x43004300u;
  return (u32x4){(w & m) | e, ((w >> 4) & m) | e, ((w >> 8) & m) | e, ((w >> 12) & m) | e};
}

// Two numbers as f16, and back.
__device__ __forceinline__ uint32_t f2h2(float a, float b) {
  return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
}
__device__ __forceinline__ float h_lo(uint32_t v) { return (float)__builtin_bit_cast(f16x2, v)[0]; }
__device__ __forceinline__ float h_hi(uint32_t v) { return (float)__builtin_bit_cast(f16x2, v)[1]; }

// silu(g) * u. exp2 and the reciprocal are the hardware's (1 ulp); the product
// under exp2 adds |g| half steps of f32. h is rounded to 11 or more bits right after.
__device__ __forceinline__ float swiglu(float g, float u) {
  const float q = __builtin_amdgcn_exp2f(-1.44269504089f * g);
  return g * __builtin_amdgcn_rcpf(1.0f + q) * u;
}

constexpr int kPassEntries = 1 << 18;  // of a pass over the experts
constexpr int kStageK = 128;           // k of a stage: two groups
// Inner up to which wide down keeps its rows in LDS: 64 rows of 512 and what goes with
// them take 77 KB, so that two work-groups share a CU's 160; 640 would leave one.
constexpr int kWideInner = 512;
// The bytes of x that a pass's 32-bit offsets reach, and an offset past them.
constexpr uint32_t kReach = 0xFFFF0000u, kNowhere = 0xFFFF8000u;

// Work-space of a pass: the plan, then what the products hand to each other.
struct MoeSpace {
  int32_t* ntiles;
  int4* tiles;     // expert, first sorted row, rows, -
  int2* perm;      // token and entry of a sorted row
  uint16_t* xs;    // [T][3][gpad(hidden)] split group sums of x
  uint16_t* xmax;  // [T][16] largest |x| of runs of 512 columns
  uint16_t* hs;    // [entries][3][gpad(inner)] split group sums of h, by sorted row
  uint16_t* h;     // [entries, inner] f16 of 2^-hexp by sorted row, or
                   // [entries][2][inner] two bf16 parts by entry (moe_few_up_kernel)
  int32_t* hexp;   // [entries] by sorted row
  float* rows;     // [entries, hidden] weighted rows of down by entry, or
                   // f16 of 2^-exps (moe_wide_down_kernel)
  int32_t* exps;   // [entries]
  uint16_t* hmax;  // [entries][8] largest |h| of a row's groups by sorted row, inner <= 512
  int32_t* counts; // [chunks of entries][experts] (moe_count_kernel)
  size_t bytes;
};

// Entries of a chunk of the two-launch plan, and those up to which one launch
// does it.
constexpr int kChunk = 4096, kPlanEntries = 8192;

// Most entries of a call whose work-groups find their rows by themselves: a
// wave holds every id.
// They and the rows' product with the sum are two launches: one token of 9 columns,
// hidden 2048, inner 512, takes 7.1 + 6.1 us, the latency of a launch and a chain of
// loads each (16 MB of weights); by a plan, tiles and a sum the call took 21.7.
constexpr int kFewEntries = 64;
// ... and the most tokens: down reads an expert's weights for each of them again.
constexpr int kFewTokens = 6;

// Groups of k columns, padded with zeros to whole 16-byte loads.
__host__ __device__ __forceinline__ int gpad(int k) { return (k / 64 + 7) & ~7; }

// Slots for tiles of `rows` rows (moe_plan_kernel).
int64_t max_tiles(int64_t entries, int experts, int rows) { return entries / rows + experts; }

// Entries from which a call goes in tiles of 64 rows (launch_moe says why): 32 an expert
// and, of its blocks of 256 columns, a work-group for most of the 512 that run side by
// side, where the tiles are the whole ones and half an expert's last.
int64_t wide_entries(int hidden, int experts) {
  const int64_t blocks = (hidden + 255) / 256, tiles = (384 + blocks - 1) / blocks;
  return std::max<int64_t>(32 * (int64_t)experts, 64 * (tiles - experts + experts / 2));
}

MoeSpace moe_space(void* base, int hidden, int inner, int experts, int64_t tokens,
                   int64_t entries) {
  MoeSpace s{};
  char* const p = static_cast<char*>(base);
  size_t at = 0;
  auto take = [&](size_t n) {
    char* const r = p + at;
    at += (n + 255) & ~(size_t)255;
    return r;
  };
  s.ntiles = reinterpret_cast<int32_t*>(take(4));
  s.tiles = reinterpret_cast<int4*>(take(max_tiles(entries, experts, 16) * sizeof(int4)));
  s.perm = reinterpret_cast<int2*>(take(entries * 8));
  s.xs = reinterpret_cast<uint16_t*>(take(tokens * 6 * gpad(hidden)));
  s.xmax = reinterpret_cast<uint16_t*>(take(tokens * 32));
  s.hs = reinterpret_cast<uint16_t*>(take(entries * 6 * gpad(inner)));
  s.h = reinterpret_cast<uint16_t*>(
      take(std::max(entries, 2 * std::min<int64_t>(entries, kFewEntries)) * inner * 2));
  s.hexp = reinterpret_cast<int32_t*>(take(entries * 4));
  // rows of long prompts are f16 (moe_wide_down_kernel), those of smaller calls f32
  const int64_t f32 =
      inner <= kWideInner ? std::min(entries, wide_entries(hidden, experts)) : entries;
  s.rows = reinterpret_cast<float*>(take(std::max(4 * f32, 2 * entries) * hidden));
  s.exps = reinterpret_cast<int32_t*>(take(entries * 4));
  s.hmax = reinterpret_cast<uint16_t*>(take(inner <= kWideInner ? entries * 16 : 0));
  s.counts = reinterpret_cast<int32_t*>(take((entries + kChunk - 1) / kChunk * experts * 4));
  s.bytes = at;
  return s;
}

// Largest value of 8 neighbouring lanes, in all of them.
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t max8(uint32_t v) {
  return max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(v)));  // lane ^ 1, ^ 2, half mirror
}

// v as three bf16 parts, v = hi + mid + lo exactly, at dst, dst + step, ...
__device__ __forceinline__ void store_split(float v, uint16_t* dst, int step) {
  const uint16_t hi = f2bf(v);
  const float q = v - bf2f(hi);
  const uint16_t mid = f2bf(q);
  dst[0] = hi;
  dst[step] = mid;
  dst[2 * step] = f2bf(q - bf2f(mid));
}

// Largest |v| of two numbers in 16 bits, in the order of their bits (infinity above
// every number, NaN above it).
__device__ __forceinline__ uint32_t max_abs2(uint32_t v) {
  return max(v & 0x7FFFu, v >> 16 & 0x7FFFu);
}

// Split group sums of x's rows, [T][3][gpad(hidden)] (not if sums is null), and the
// largest |x| of every 512 columns, [T][16]. A lane takes 8 of a group's 64 columns, 8
// lanes a group, a wave 8 groups; a thread of a padded group stores zeros. i: the
// thread's number.
__device__ __forceinline__ void moe_row_sums(const uint16_t* __restrict__ x, int64_t xs, int T,
                                             int hidden, uint16_t* __restrict__ sums,
                                             uint16_t* __restrict__ xmax, int64_t i) {
  const int gp = gpad(hidden);
  const int64_t t = i / (8 * gp);
  const int c = (int)(i - t * 8 * gp);  // 8-column chunk of the row
  if (t >= T) return;
  float v = 0.f;
  uint32_t m = 0;
  if (8 * c < hidden) {
    const u32x4 q = *reinterpret_cast<const u32x4*>(x + t * xs + 8 * c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v += bf_lo(q[e]) + bf_hi(q[e]);
      m = max(m, max_abs2(q[e]));
    }
  }
  // 8 lanes, a row of 16, then rows 0 -> 1, 2 -> 3 and 1 -> 2, 3: lane 63 has all
  m = max_dpp<0x143>(max_dpp<0x142>(max_dpp<0x128>(max8(m))));
  if ((c & 63) == 63) xmax[t * 16 + c / 64] = (uint16_t)m;
  if (!sums) return;
  v = sum8(v);
  if ((c & 7) == 0) store_split(v, sums + t * 3 * gp + c / 8, gp);
}

struct RowMax {
  u32x4 v[2];  // 16 maxima
};
__device__ __forceinline__ RowMax load_row_max(const uint16_t* xmax, int64_t token) {
  const u32x4* const p = reinterpret_cast<const u32x4*>(xmax + token * 16);
  return {{p[0], p[1]}};
}
// The exponent of h's power of two for a row of x and the expert's bounds of gate and
// up: |h| 2^-exponent < 2^15. It stays where 2^exponent and 2^-exponent are f32 numbers:
// h, an f32 number itself, is below 2^(113 + 15), and where the bound lets it be raised
// by 2^126 only, it is below 2^(15 - 126).
__device__ __forceinline__ int row_exponent(const RowMax& xm, int hidden, const float (&bound)[2]) {
  const int n = gpad(hidden) >> 3;
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if (2 * q < n) m = max(m, xm.v[q >> 2][q & 3] & 0xFFFFu);
    if (2 * q + 1 < n) m = max(m, xm.v[q >> 2][q & 3] >> 16);
  }
  const int e = __builtin_amdgcn_frexp_expf(bound[0]) + __builtin_amdgcn_frexp_expf(bound[1]) +
                2 * __builtin_amdgcn_frexp_expf(__uint_as_float(m << 16)) - 15;
  return max(-126, min(e, 113));
}

// The plan: work-group e sorts expert e's entries, in entry order, behind those
// of the experts before it, and lists its tiles. It counts the entries of lower
// experts and its own by itself, so that one launch without atomics does it.
// Expert e's tiles start at slot (entries before it) / rows + e: never fewer
// slots than tiles, the ones left over marked empty (rows = 0).
// Work-groups from `experts` on form the split group sums and maxima of x's rows
// (moe_row_sums) beside it. 4 to 5 us up to 8192 entries: a launch and two rounds of
// loads.
constexpr int kPlanThreads = 1024;
typedef int i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
__global__ __launch_bounds__(kPlanThreads) void moe_plan_kernel(MoeArgs a, int rows, MoeSpace s) {
  constexpr int W = kPlanThreads / 64;
  __shared__ int lower[W], own[W];
  const int32_t* const ids = a.ids;
  const int entries = a.T * a.k, k = a.k, experts = a.experts;
  if (blockIdx.x >= (uint32_t)experts) {
    moe_row_sums(a.x, a.xs, a.T, a.hidden, s.xs, s.xmax,
                 (int64_t)(blockIdx.x - experts) * kPlanThreads + threadIdx.x);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t e = blockIdx.x;
  // a wave takes a run of entries, 4 a lane at a time, so that they keep their order
  const int run = ((entries + W - 1) / W + 255) & ~255;
  const int i0 = wave * run, i1 = min(entries, i0 + run);
  auto load = [&](int i, int (&v)[4]) {
    if (i + 4 <= i1) {
      const i32x4_a4 q = *reinterpret_cast<const i32x4_a4*>(ids + i);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = q[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = i + c < i1 ? ids[i + c] : -1;
    }
  };
  int lo = 0, mine = 0;
#pragma unroll 4
  for (int i = i0 + 4 * lane; i < i1; i += 256) {
    int v[4];
    load(i, v);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      lo += (uint32_t)v[c] < e;
      mine += (uint32_t)v[c] == e;
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    lo += __shfl_xor(lo, off, 64);
    mine += __shfl_xor(mine, off, 64);
  }
  if (lane == 0) {
    lower[wave] = lo;
    own[wave] = mine;
  }
  __syncthreads();
  int before = 0, n = 0, at = 0;
  for (int w = 0; w < W; ++w) {
    before += lower[w];
    at += w < wave ? own[w] : 0;
    n += own[w];
  }
  const int t0 = before / rows + (int)e, t1 = (before + n) / rows + (int)e + 1;
  if ((int)e == experts - 1 && tid == 0) *s.ntiles = t1;
  for (int i = tid; i < t1 - t0; i += kPlanThreads)
    s.tiles[t0 + i] = make_int4((int)e, before + rows * i, max(0, min(rows, n - rows * i)), 0);
  if (mine == 0) return;
  at += before;
  for (int i = i0 + 4 * lane; i - 4 * lane < i1; i += 256) {
    int v[4];
    load(i, v);
    int below = 0, all = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint64_t b = __ballot((uint32_t)v[c] == e);
      below += __popcll(b & ((1ull << lane) - 1));
      all += __popcll(b);
    }
    if (all == 0) continue;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if ((uint32_t)v[c] == e) s.perm[at + below++] = make_int2((i + c) / k, i + c);
    at += all;
  }
}

// The plan of many entries in two launches. First a work-group per chunk of
// entries counts them by expert; others form the rows' sums.
__global__ __launch_bounds__(kPlanThreads) void moe_count_kernel(MoeArgs a, int chunks, MoeSpace s) {
  extern __shared__ int cnt[];
  if (blockIdx.x >= (uint32_t)chunks) {
    moe_row_sums(a.x, a.xs, a.T, a.hidden, s.xs, s.xmax,
                 (int64_t)(blockIdx.x - chunks) * kPlanThreads + threadIdx.x);
    return;
  }
  for (int e = threadIdx.x; e < a.experts; e += kPlanThreads) cnt[e] = 0;
  __syncthreads();
  const int i1 = min(a.T * a.k, (int)(blockIdx.x + 1) * kChunk);
  for (int i = blockIdx.x * kChunk + threadIdx.x; i < i1; i += kPlanThreads) {
    const int id = a.ids[i];
    if ((uint32_t)id < (uint32_t)a.experts) atomicAdd(&cnt[id], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kPlanThreads)
    s.counts[(int64_t)blockIdx.x * a.experts + e] = cnt[e];
}

// Then a work-group per chunk places its entries behind those of lower experts
// and of its expert in the chunks before, and writes its share of the tile list.
// Inside a chunk an expert's entries take their places in any order: a row's
// sums do not depend on where it stands. 147,456 entries of 16,384 rows: 18.5 us, most
// of it reading x for the sums and maxima, and 9.6; in one launch as above 58.
__global__ __launch_bounds__(kPlanThreads) void moe_place_kernel(MoeArgs a, int rows, MoeSpace s) {
  extern __shared__ int lds[];
  __shared__ int wsum[kPlanThreads / 64];
  const int E = a.experts, chunks = gridDim.x, chunk = blockIdx.x;
  int* const before = lds;   // entries of lower experts
  int* const at = lds + E;   // the chunk's next place of an expert
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int epp = (E + kPlanThreads - 1) / kPlanThreads;  // experts of a thread, in a run
  int mine = 0;
  for (int e = tid * epp; e < min(E, (tid + 1) * epp); ++e) {
    int n = 0, o = 0;
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) {
      const int v = s.counts[(int64_t)c * E + e];
      n += v;
      o += c < chunk ? v : 0;
    }
    before[e] = n;
    at[e] = o;
    mine += n;
  }
  int run = mine;  // inclusive over the wave, then over the waves
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int v = __shfl_up(run, off, 64);
    run += lane >= off ? v : 0;
  }
  if (lane == 63) wsum[wave] = run;
  __syncthreads();
  run -= mine;
  for (int w = 0; w < wave; ++w) run += wsum[w];
  for (int e = tid * epp; e < min(E, (tid + 1) * epp); ++e) {
    const int n = before[e];
    before[e] = run;
    at[e] += run;
    run += n;
  }
  __syncthreads();
  int total = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) total += wsum[w];
  // slots as in moe_plan_kernel: expert e's from before / rows + e on
  const int slots = total / rows + E, share = (slots + chunks - 1) / chunks;
  if (chunk == 0 && tid == 0) *s.ntiles = slots;
  for (int t = chunk * share + tid; t < min(slots, (chunk + 1) * share); t += kPlanThreads) {
    int lo = 0, hi = E - 1;  // the last expert whose slots start at t or before
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if (before[m] / rows + m <= t)
        lo = m;
      else
        hi = m - 1;
    }
    const int n = (lo + 1 < E ? before[lo + 1] : total) - before[lo];
    const int i = t - before[lo] / rows - lo;
    s.tiles[t] = make_int4(lo, before[lo] + rows * i, max(0, min(rows, n - rows * i)), 0);
  }
  const int i1 = min(a.T * a.k, (chunk + 1) * kChunk);
  for (int i = chunk * kChunk + tid; i < i1; i += kPlanThreads) {
    const int id = a.ids[i];
    if ((uint32_t)id < (uint32_t)E) s.perm[atomicAdd(&at[id], 1)] = make_int2(i / a.k, i);
  }
}

// ---- very few entries: no plan ----

// NS stages p0, p0 + step, ... of a 16-row fragment: its weights, scales and
// biases (stages past P: the last one again; their x is zero).
template <int NS>
struct Frag {
  u32x4 w[NS];
  uint32_t s[NS], b[NS];
  __device__ __forceinline__ void load(const u32x4* wp, const uint32_t* sb, int P, int p0,
                                       int step) {
    const int lane = threadIdx.x & 63, r16 = lane & 15;
#pragma unroll
    for (int q = 0; q < NS; ++q) {
      const int p = min(p0 + step * q, P - 1);
      w[q] = __builtin_nontemporal_load(wp + p * 64 + lane);
      s[q] = __builtin_nontemporal_load(sb + p * 32 + r16);
      b[q] = __builtin_nontemporal_load(sb + p * 32 + 16 + r16);
    }
  }
};

// The same stages of 16 rows of x; lane (r16, c4) holds row r16 (row null:
// zeros). Sums of a group: xg rows 4 c4 + i.
template <int NS>
struct Rows {
  u32x4 x[NS][4];
  __device__ __forceinline__ void load(const uint16_t* row, int P, int p0, int step) {
    const int c4 = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int q = 0; q < NS; ++q) {
      const int p = p0 + step * q;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        x[q][h] = (u32x4){0u, 0u, 0u, 0u};
        if (row && p < P) x[q][h] = *reinterpret_cast<const u32x4*>(row + 128 * p + 32 * h + 8 * c4);
      }
    }
  }
};

// T[f] += x . w of NF fragments over NS stages. x is the MFMA A operand: a
// lane ends with rows 4 c4 + i, column r16 of each fragment, so that one scale
// and one offset per group serve all of its sums.
template <int NF, int NS>
__device__ __forceinline__ void product(const Rows<NS>& x, const Frag<NS> (&f)[NF], uint32_t nib,
                                        f32x4 (&T)[NF]) {
  const u32x4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < NS; ++q) {
    __builtin_amdgcn_sched_barrier(0);  // one stage's operands at a time
#pragma unroll
    for (int gl = 0; gl < 2; ++gl) {
      f32x4 xg = mfma(x.x[q][2 * gl], ones, zero);
      xg = mfma(x.x[q][2 * gl + 1], ones, xg);
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        f32x4 d = mfma(x.x[q][2 * gl], unpack_w(f[i].w[q][2 * gl], nib), zero);
        d = mfma(x.x[q][2 * gl + 1], unpack_w(f[i].w[q][2 * gl + 1], nib), d);
        const float sc = gl ? bf_hi(f[i].s[q]) : bf_lo(f[i].s[q]);
        const float of = fmaf(-128.0f, sc, gl ? bf_hi(f[i].b[q]) : bf_lo(f[i].b[q]));
#pragma unroll
        for (int r = 0; r < 4; ++r) T[i][r] = fmaf(sc, d[r], fmaf(of, xg[r], T[i][r]));
      }
    }
  }
}

// h by entry, as two bf16 parts (16 bits): the second is one more row of down's
// product, which has 16 of them for one. Work-group (entry u, 16 inner columns), four
// waves, wave w over the stages 4 w .. 4 w + 3 (and on from 16 stages ahead), added in
// wave order.
// It takes every row of the expert that entry u names first; a later entry of
// the same expert has nothing to do.
__global__ __launch_bounds__(256) void moe_few_up_kernel(MoeArgs a, uint16_t* __restrict__ h) {
  __shared__ f32x4 part[4][2][64];
  const int blocks = a.inner / 16, entries = a.T * a.k;
  const int u = blockIdx.x / blocks, j = blockIdx.x - u * blocks;
  const int lane = threadIdx.x & 63, r16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = lane < entries ? a.ids[lane] : -1;
  const int e = __builtin_amdgcn_readlane(id, u);
  const uint64_t hits = __ballot(id == e);
  if ((uint32_t)e >= (uint32_t)a.experts || (hits & ((1ull << u) - 1)) != 0) return;
  const int n = __popcll(hits);
  // lane r receives the r-th entry of the expert (the others push to lane 63, which
  // is read only where it is itself the 64th)
  const int rank = id == e ? __popcll(hits & ((1ull << lane) - 1)) : 63;
  const int mine = __builtin_amdgcn_ds_permute(rank << 2, lane);
  const int P = a.hidden >> 7;
  const int64_t f0 = ((int64_t)e * blocks + j) * 2 * P;
  const u32x4* const wp = static_cast<const u32x4*>(a.w1) + f0 * 64;
  const uint32_t* const sb = a.sb1 + f0 * 32;
  uint32_t nib = 0x000F000Fu;
  asm volatile("" : "+v"(nib));
  for (int m0 = 0; m0 < n; m0 += 16) {
    const int en = __shfl(mine, m0 + r16, 64);
    const uint16_t* const row = m0 + r16 < n ? a.x + (int64_t)(en / a.k) * a.xs : nullptr;
    f32x4 T[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int p = 4 * wave; p < P; p += 16) {
      Frag<4> f[2];
      Rows<4> x;
#pragma unroll
      for (int i = 0; i < 2; ++i) f[i].load(wp + (int64_t)i * P * 64, sb + (int64_t)i * P * 32, P, p, 1);
      x.load(row, P, p, 1);
      product<2, 4>(x, f, nib, T);
    }
    part[wave][0][lane] = T[0];
    part[wave][1][lane] = T[1];
    __syncthreads();
    // thread (element i of lane l): row 4 (l / 16) + i, column l % 16
    const int l = threadIdx.x >> 2, i = threadIdx.x & 3, m = m0 + 4 * (l >> 4) + i;
    const int em = __shfl(mine, m, 64);
    float g = 0.f, up = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      g += part[w][0][l][i];
      up += part[w][1][l][i];
    }
    if (m < n) {
      const float v = swiglu(g, up);
      const uint16_t hi = f2bf(v);
      uint16_t* const o = h + 2 * (int64_t)em * a.inner + 16 * j + (l & 15);
      o[0] = hi;
      o[a.inner] = f2bf(v - bf2f(hi));
    }
    __syncthreads();
  }
}

// Down and the sum over a token's columns in one. Work-group
// (token, 16 columns), a wave per column of ids (rounds of 16), added in order.
__global__ __launch_bounds__(1024) void moe_few_down_kernel(MoeArgs a,
                                                              const uint16_t* __restrict__ h) {
  __shared__ float part[16][16];
  const int blocks = a.hidden / 16, t = blockIdx.x / blocks, j = blockIdx.x - t * blocks;
  const int lane = threadIdx.x & 63, r16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int P = a.inner >> 7;
  uint32_t nib = 0x000F000Fu;
  asm volatile("" : "+v"(nib));
  float y = 0.f;
  for (int c0 = 0; c0 < a.k; c0 += waves) {
    const int c = c0 + wave, en = t * a.k + c;
    const int e = c < a.k ? __builtin_amdgcn_readfirstlane(a.ids[en]) : -1;
    f32x4 T[1] = {{0.f, 0.f, 0.f, 0.f}};
    if ((uint32_t)e < (uint32_t)a.experts) {
      const int64_t f0 = ((int64_t)e * blocks + j) * P;
      const uint16_t* const row = r16 < 2 ? h + (2 * (int64_t)en + r16) * a.inner : nullptr;
      for (int p = 0; p < P; p += 4) {
        Rows<4> x;
        Frag<4> f[1];
        f[0].load(static_cast<const u32x4*>(a.w2) + f0 * 64, a.sb2 + f0 * 32, P, p, 1);
        x.load(row, P, p, 1);
        product<1, 4>(x, f, nib, T);
      }
      T[0][0] = (T[0][0] + T[0][1]) * a.weights[en];
    }
    if (lane < 16) part[wave][lane] = T[0][0];
    __syncthreads();
    if (threadIdx.x < 16)
      for (int w = 0; w < min(waves, a.k - c0); ++w) y += part[w][threadIdx.x];
    __syncthreads();
  }
  if (threadIdx.x < 16) a.out[(int64_t)t * a.os + 16 * j + threadIdx.x] = f2bf(y);
}

// s_waitcnt lgkmcnt(0), and vmcnt(N) below (gfx9 encodings, the other counters
// at their maximum)
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xC07F); }

// v 2^e
__device__ __forceinline__ f32x4 scaled(f32x4 v, int e) {
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = ldexpf(v[r], e);
  return v;
}

// ---- tiles ----

template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// A tile of 16 MW rows against 128 columns (8 fragments); four waves in a row,
// each with all rows and two fragments. The weights are the MFMA A operand, so a
// lane ends with four consecutive columns of one row.
// Per stage of 128 k the rows go to LDS by DMA, 16-byte chunk c of row r at
// chunk c ^ (r % 16) (operand reads without conflicts), as do the fragments'
// scales; the weights go to registers; all of them R - 1 stages ahead. The ring's
// slots are arrays of their own, so that the compiler can tell copies into one
// from reads of another.
// The offsets' sum over the groups, sum_g (b_g - 128 s_g) X_g, is a short MFMA
// product at the end: X_g as three bf16 parts (exact), b and s as stored.
//   UP: rows are gathered tokens of x, the fragments gate and up in turn: a wave
//     ends with gate and up of the same 16 columns and stores h; the work-group's
//     64 columns are one group of down's input, whose split sums it stores.
//   else: rows of h, and the weighted rows of down go to their entries.
// Bound by the weights' bytes and the loads' latency: 317 tokens of 9 columns, hidden
// 2048, inner 512, 257 experts (11 rows each): up 67 us (303 MB, 4.5 TB/s), down 43
// (152 MB, 3.5 TB/s).
template <int MW, bool UP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4, 8))) void moe_tile_kernel(
    MoeArgs a, MoeSpace s) {
  constexpr int MT = 16 * MW, XROW = kStageK * 2, R = 3;
  constexpr int LB = MW + 3;  // loads of a stage
  __shared__ __align__(16) uint8_t xl0[MT * XROW], xl1[MT * XROW], xl2[MT * XROW];
  __shared__ __align__(16) uint8_t sl0[4 * 256], sl1[4 * 256], sl2[4 * 256];
  __shared__ float gsum[UP ? 4 : 1][MT];
  const int K = UP ? a.hidden : a.inner, N = UP ? 2 * a.inner : a.hidden;
  const int P = K >> 7, blocks = N >> 7;
  // an XCD (work-groups L % 8) takes a run of the tiles, all columns of a tile
  // side by side
  const int n = *s.ntiles * blocks, per = (n + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || idx >= n) return;
  const int tile = idx / blocks, cb = idx - tile * blocks;
  int4 tl = s.tiles[tile];
  tl.x = __builtin_amdgcn_readfirstlane(tl.x);
  tl.y = __builtin_amdgcn_readfirstlane(tl.y);
  tl.z = __builtin_amdgcn_readfirstlane(tl.z);
  if (tl.z == 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, c4 = lane >> 4;

  const int64_t f0 = (int64_t)tl.x * (N >> 4) + 8 * cb;  // first fragment of the work-group
  const u32x4* const wp = static_cast<const u32x4*>(UP ? a.w1 : a.w2) + f0 * P * 64;
  const uint32_t* const sb = (UP ? a.sb1 : a.sb2) + f0 * P * 32;
  const uint16_t* const xbase = UP ? a.x : s.h + (int64_t)tl.y * a.inner;
  uint32_t xvo[MW];
#pragma unroll
  for (int j = 0; j < MW; ++j) {
    const int r = 4 * (wave + 4 * j) + c4, src = min(r, tl.z - 1);
    const int64_t at = UP ? (int64_t)s.perm[tl.y + src].x * a.xs : (int64_t)src * a.inner;
    xvo[j] = (uint32_t)(at * 2) + 16 * (r16 ^ (r & 15));
  }
  const int wvo = (wave * 2 * P * 64 + lane) * 16;
  // scale copy: lane L -> fragment (L / 16) % 2 of the wave, dword L % 16
  const int svo = (wave * 2 + (c4 & 1)) * P * 128 + 4 * r16;

  u32x4 wr[R][2];
  auto xbuf = [&](auto slot) -> uint8_t* {
    constexpr int S = decltype(slot)::value;
    return S == 0 ? xl0 : S == 1 ? xl1 : xl2;
  };
  auto sbuf = [&](auto slot) -> uint8_t* {
    constexpr int S = decltype(slot)::value;
    return (S == 0 ? sl0 : S == 1 ? sl1 : sl2) + wave * 256;
  };
  // stage p's loads into ring slot S (none of a stage past the last)
  auto batch = [&](int p, auto slot) {
    constexpr int S = decltype(slot)::value;
    const int in = __builtin_amdgcn_readfirstlane(p < P ? -1 : 0);
    const __amdgpu_buffer_rsrc_t xrs =
        __builtin_amdgcn_make_buffer_rsrc((void*)xbase, (short)0, in, 0x00020000);
    const __amdgpu_buffer_rsrc_t wrs =
        __builtin_amdgcn_make_buffer_rsrc((void*)wp, (short)0, in & (8 * P * 1024), 0x00020000);
    const __amdgpu_buffer_rsrc_t srs =
        __builtin_amdgcn_make_buffer_rsrc((void*)sb, (short)0, in & (8 * P * 128), 0x00020000);
#pragma unroll
    for (int j = 0; j < MW; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xrs, (void __attribute__((address_space(3)))*)(xbuf(slot) + 4 * (wave + 4 * j) * XROW),
          16, (int)xvo[j], p * XROW, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      wr[S][i] = __builtin_amdgcn_raw_buffer_load_b128(wrs, wvo, (i * P + p) * 1024, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        srs, (void __attribute__((address_space(3)))*)sbuf(slot), 4, svo, p * 128, 0, 0);
  };
  // all but the youngest B stages have landed, in every wave
  auto landed = [&](auto behind) {
    wait_vm<decltype(behind)::value * LB>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "global");
  };
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 T[2][MW];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int u = 0; u < MW; ++u) T[i][u] = zero;
  uint32_t nib = 0x000F000Fu;
  asm volatile("" : "+v"(nib));

  auto compute = [&](auto slot) {
    constexpr int S = decltype(slot)::value;
    const uint8_t* const cur = xbuf(slot);
    u32x4 sv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      sv[i] = *reinterpret_cast<const u32x4*>(sbuf(slot) + i * 64 + c4 * 16);
#pragma unroll
    for (int gl = 0; gl < 2; ++gl) {
      u32x4 A[2][2];
      float sc[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        A[i][0] = unpack_w<!UP>(wr[S][i][2 * gl], nib);
        A[i][1] = unpack_w<!UP>(wr[S][i][2 * gl + 1], nib);
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[i][r] = gl ? bf_hi(sv[i][r]) : bf_lo(sv[i][r]);
      }
#pragma unroll
      for (int u = 0; u < MW; ++u) {
        u32x4 X[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          X[h] = *reinterpret_cast<const u32x4*>(
              &cur[(u * 16 + r16) * XROW + (((8 * gl + 4 * h + c4) ^ r16) << 4)]);
        f32x4 d[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) d[i] = mfma<!UP>(A[i][0], X[0], zero);
#pragma unroll
        for (int i = 0; i < 2; ++i) d[i] = mfma<!UP>(A[i][1], X[1], d[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) T[i][u][r] = fmaf(sc[i][r], d[i][r], T[i][u][r]);
      }
    }
  };
  // Whole turns of the ring, then up to R - 1 stages more. The turns' body has no
  // branch: a stage past the last one is loaded through an empty resource.
  auto step = [&](int p, auto slot) {
    constexpr int S = decltype(slot)::value;
    batch(p + R - 1, std::integral_constant<int, (S + R - 1) % R>{});
    __builtin_amdgcn_sched_barrier(0);
    compute(slot);
    landed(std::integral_constant<int, R - 2>{});
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;
  // `landed` counts loads: all of stage 0 go out before stage 1's first
  batch(0, S0{});
  __builtin_amdgcn_sched_barrier(0);
  batch(1, S1{});
  __builtin_amdgcn_sched_barrier(0);
  landed(std::integral_constant<int, R - 2>{});

  // rows' sums, and where down's rows go
  const int gp = gpad(K), go = gp >> 3;
  const uint16_t* xg[MW];
  int en[MW];
  RowMax xm[UP ? MW : 1];
  float bound[2];
#pragma unroll
  for (int u = 0; u < MW; ++u) {
    const int row = tl.y + min(u * 16 + r16, tl.z - 1);
    const int2 pe = s.perm[row];
    xg[u] = UP ? s.xs + (int64_t)pe.x * 3 * gp : s.hs + (int64_t)row * 3 * gp;
    en[u] = pe.y;
    if constexpr (UP) xm[u] = load_row_max(s.xmax, pe.x);
  }
  if constexpr (UP)
    for (int i = 0; i < 2; ++i) bound[i] = a.bound[i * a.experts + tl.x];
  int p = 0;
#pragma nounroll
  for (; p + R <= P; p += R) {
    step(p, S0{});
    step(p + 1, S1{});
    step(p + 2, S2{});
  }
  if (p < P) {
    compute(S0{});
    landed(std::integral_constant<int, 0>{});
    if (p + 1 < P) compute(S1{});
  }
  wait_vm<0>();  // no copy is left behind

  // The offsets' sum. A row's sums are [hi | mid | lo][gp]: octet o of the row is
  // part o / go of groups 8 (o % go) .., and a product takes four octets, one a
  // lane group.
  float wt[MW];
  int he[MW];  // exponents of h's rows
#pragma unroll
  for (int u = 0; u < MW; ++u) {
    if constexpr (UP) {
      he[u] = row_exponent(xm[u], a.hidden, bound);
    } else {
      wt[u] = a.weights[en[u]];
      he[u] = s.hexp[tl.y + min(u * 16 + r16, tl.z - 1)];
    }
  }
#pragma nounroll
  for (int jb = 0; 4 * jb < 3 * go; ++jb) {
    const int o = 4 * jb + c4, oc = o < go ? o : o < 2 * go ? o - go : o - 2 * go;
    u32x4 as[2], ab[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int ps = 4 * oc + q;
        const bool in = o < 3 * go && ps < P;
        const uint32_t* const sq = sb + ((wave * 2 + i) * P + (in ? ps : 0)) * 32 + r16;
        as[i][q] = in ? sq[0] : 0u;
        ab[i][q] = in ? sq[16] : 0u;
      }
#pragma unroll
    for (int u = 0; u < MW; ++u) {
      const u32x4 xp = *reinterpret_cast<const u32x4*>(xg[u] + 8 * (o < 3 * go ? o : 0));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x4 d = mfma(as[i], xp, zero);
        T[i][u] = mfma(ab[i], xp, T[i][u]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          T[i][u][r] = fmaf(UP ? -kOffsetX : -kOffsetH, d[r], T[i][u][r]);
      }
    }
  }

  if constexpr (UP) {
    const int col = 64 * cb + 16 * wave + 4 * c4;
#pragma unroll
    for (int u = 0; u < MW; ++u) {
      const int m = u * 16 + r16;
      const float sc = ldexpf(1.0f, -he[u]);
      const uint32_t lo =
          f2h2(sc * swiglu(T[0][u][0], T[1][u][0]), sc * swiglu(T[0][u][1], T[1][u][1]));
      const uint32_t hi =
          f2h2(sc * swiglu(T[0][u][2], T[1][u][2]), sc * swiglu(T[0][u][3], T[1][u][3]));
      if (m < tl.z) {
        *reinterpret_cast<u32x2*>(s.h + (int64_t)(tl.y + m) * a.inner + col) = (u32x2){lo, hi};
        if (cb == 0 && wave == 0 && c4 == 0) s.hexp[tl.y + m] = he[u];
      }
      float v = (h_lo(lo) + h_hi(lo)) + (h_lo(hi) + h_hi(hi));
      v += __shfl_xor(v, 16, 64);
      v += __shfl_xor(v, 32, 64);
      if (c4 == 0) gsum[wave][m] = v;
    }
    lds_barrier();
    if (tid < tl.z) {
      const int gi = gpad(a.inner);
      uint16_t* const dst = s.hs + (int64_t)(tl.y + tid) * 3 * gi;
      store_split((gsum[0][tid] + gsum[1][tid]) + (gsum[2][tid] + gsum[3][tid]), dst + cb, gi);
      if (cb == blocks - 1)  // the padded groups
        for (int g = blocks; g < gi; ++g) store_split(0.f, dst + g, gi);
    }
  } else {
#pragma unroll
    for (int u = 0; u < MW; ++u) {
      if (u * 16 + r16 >= tl.z) continue;
      float* const o = s.rows + (int64_t)en[u] * a.hidden + 128 * cb + 32 * wave + 4 * c4;
#pragma unroll
      for (int i = 0; i < 2; ++i) *reinterpret_cast<f32x4*>(o + 16 * i) = scaled(wt[u] * T[i][u], he[u]);
    }
  }
}

// moe_tile_kernel for up to 16 rows, where the weights' stream is the work:
// 64 columns a work-group (small ones fill the chip evenly), KS pairs of waves each
// over a part of the stages (a wave's stages run one after the other, so that a
// small call takes as long as one wave's), the groups' sums of x from products
// against ones instead of beforehand, and the offsets applied with the scales. Rows
// past the tile's are not read: their copies are out of the buffer's range, which
// gives zeros. Bound by the weights' bytes: 64 tokens of 9 columns, hidden 2048, inner
// 512, 257 experts: up 45.5 us at 5.8 TB/s, down 26.6 at 4.9.
template <int KS, bool UP>
__global__ __launch_bounds__(128 * KS) __attribute__((amdgpu_waves_per_eu(4, 8))) void
    moe_stream_kernel(MoeArgs a, MoeSpace s) {
  constexpr int XROW = kStageK * 2, R = 3, LB = 2 + 2 + 1;
  __shared__ __align__(16) uint8_t xl0[KS][16 * XROW], xl1[KS][16 * XROW], xl2[KS][16 * XROW];
  __shared__ __align__(16) uint8_t sl0[512 * KS], sl1[512 * KS], sl2[512 * KS];
  const int K = UP ? a.hidden : a.inner, N = UP ? 2 * a.inner : a.hidden;
  const int P = K >> 7, blocks = N >> 6;
  const int n = *s.ntiles * blocks, per = (n + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || idx >= n) return;
  const int tile = idx / blocks, cb = idx - tile * blocks;
  int4 tl = s.tiles[tile];
  tl.x = __builtin_amdgcn_readfirstlane(tl.x);
  tl.y = __builtin_amdgcn_readfirstlane(tl.y);
  tl.z = __builtin_amdgcn_readfirstlane(tl.z);
  if (tl.z == 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, c4 = lane >> 4;
  const int cw = wave & 1, kw = wave >> 1;  // column pair, part of the stages
  // the part's stages: p0 + (0 .. mine - 1), mine or one less for every part
  const int least = P / KS, more = P - least * KS;
  const int p0 = kw * least + min(kw, more), mine = least + (kw < more);

  const int64_t f0 = (int64_t)tl.x * (N >> 4) + 4 * cb + 2 * cw;  // the wave's first fragment
  const u32x4* const wp = static_cast<const u32x4*>(UP ? a.w1 : a.w2) + f0 * P * 64;
  const uint32_t* const sb = (UP ? a.sb1 : a.sb2) + f0 * P * 32;
  const uint16_t* const xbase = UP ? a.x : s.h + (int64_t)tl.y * a.inner;
  uint32_t xvo[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 4 * (cw + 2 * j) + c4;
    xvo[j] = kNowhere;
    if (r < tl.z) {
      const int64_t at = UP ? (int64_t)s.perm[tl.y + r].x * a.xs : (int64_t)r * a.inner;
      xvo[j] = (uint32_t)(at * 2) + 16 * (r16 ^ (r & 15));
    }
  }
  // a row's place for the results: the tile's sorted row (up) or its entry
  const int m = min(r16, tl.z - 1);
  const int2 pe = s.perm[tl.y + m];
  const int en = pe.y;
  const float wt = UP ? 0.f : a.weights[en];
  const int hexp = UP ? 0 : s.hexp[tl.y + m];
  const int svo = (lane >> 5) * P * 128 + 4 * (lane & 31);  // fragment, dword
  u32x4 wr[R][2];
  auto xbuf = [&](auto slot) -> uint8_t* {
    constexpr int S = decltype(slot)::value;
    return (S == 0 ? xl0 : S == 1 ? xl1 : xl2)[kw];
  };
  auto sbuf = [&](auto slot) -> uint8_t* {
    constexpr int S = decltype(slot)::value;
    return (S == 0 ? sl0 : S == 1 ? sl1 : sl2) + wave * 256;
  };
  auto batch = [&](int p, auto slot) {
    constexpr int S = decltype(slot)::value;
    const int in = __builtin_amdgcn_readfirstlane(p < mine ? -1 : 0);
    const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)xbase, (short)0, in & (int)kReach, 0x00020000);
    const __amdgpu_buffer_rsrc_t wrs =
        __builtin_amdgcn_make_buffer_rsrc((void*)wp, (short)0, in & (2 * P * 1024), 0x00020000);
    const __amdgpu_buffer_rsrc_t srs =
        __builtin_amdgcn_make_buffer_rsrc((void*)sb, (short)0, in & (2 * P * 128), 0x00020000);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xrs, (void __attribute__((address_space(3)))*)(xbuf(slot) + 4 * (cw + 2 * j) * XROW),
          16, (int)xvo[j], (p0 + p) * XROW, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)  // read once: nontemporal
      wr[S][i] = __builtin_amdgcn_raw_buffer_load_b128(wrs, lane * 16, (i * P + p0 + p) * 1024, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        srs, (void __attribute__((address_space(3)))*)sbuf(slot), 4, svo, (p0 + p) * 128, 0, 0);
  };
  auto landed = [&](auto behind) {
    wait_vm<decltype(behind)::value * LB>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "global");
  };
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const uint32_t one2 = UP ? 0x3F803F80u : 0x3C003C00u;
  const u32x4 ones = {one2, one2, one2, one2};
  f32x4 T[2] = {zero, zero};
  uint32_t nib = 0x000F000Fu;
  asm volatile("" : "+v"(nib));
  auto compute = [&](auto slot) {
    constexpr int S = decltype(slot)::value;
    const uint8_t* const cur = xbuf(slot);
    u32x4 sv[2], bv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sv[i] = *reinterpret_cast<const u32x4*>(sbuf(slot) + i * 128 + c4 * 16);
      bv[i] = *reinterpret_cast<const u32x4*>(sbuf(slot) + i * 128 + 64 + c4 * 16);
    }
#pragma unroll
    for (int gl = 0; gl < 2; ++gl) {
      u32x4 X[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        X[h] = *reinterpret_cast<const u32x4*>(
            &cur[r16 * XROW + (((8 * gl + 4 * h + c4) ^ r16) << 4)]);
      f32x4 xg = mfma<!UP>(ones, X[0], zero);
      xg = mfma<!UP>(ones, X[1], xg);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4 d = mfma<!UP>(unpack_w<!UP>(wr[S][i][2 * gl], nib), X[0], zero);
        d = mfma<!UP>(unpack_w<!UP>(wr[S][i][2 * gl + 1], nib), X[1], d);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float sc = gl ? bf_hi(sv[i][r]) : bf_lo(sv[i][r]);
          const float of =
              fmaf(UP ? -kOffsetX : -kOffsetH, sc, gl ? bf_hi(bv[i][r]) : bf_lo(bv[i][r]));
          T[i][r] = fmaf(sc, d[r], fmaf(of, xg[0], T[i][r]));
        }
      }
    }
  };
  auto step = [&](int p, auto slot) {
    constexpr int S = decltype(slot)::value;
    batch(p + R - 1, std::integral_constant<int, (S + R - 1) % R>{});
    __builtin_amdgcn_sched_barrier(0);
    compute(slot);
    landed(std::integral_constant<int, R - 2>{});
  };
  using S0 = std::integral_constant<int, 0>;
  using S1 = std::integral_constant<int, 1>;
  using S2 = std::integral_constant<int, 2>;
  // `landed` counts loads: all of stage 0 go out before stage 1's first
  batch(0, S0{});
  __builtin_amdgcn_sched_barrier(0);
  batch(1, S1{});
  __builtin_amdgcn_sched_barrier(0);
  landed(std::integral_constant<int, R - 2>{});
  RowMax xm;  // used behind the stages
  float bound[2];
  if constexpr (UP) {
    xm = load_row_max(s.xmax, pe.x);
    for (int i = 0; i < 2; ++i) bound[i] = a.bound[i * a.experts + tl.x];
  }
  int p = 0;
#pragma nounroll
  for (; p + R <= least; p += R) {
    step(p, S0{});
    step(p + 1, S1{});
    step(p + 2, S2{});
  }
  batch(p + 2, S2{});
  if (p < mine) compute(S0{});
  landed(std::integral_constant<int, 0>{});
  if (p + 1 < mine) compute(S1{});
  if (p + 2 < mine) compute(S2{});

  if constexpr (KS > 1) {  // the parts' sums, added in order
    lds_barrier();         // the slots are free once every wave is here
    f32x4* const part = reinterpret_cast<f32x4*>(xl0);
    if (kw > 0)
#pragma unroll
      for (int i = 0; i < 2; ++i) part[((kw - 1) * 4 + 2 * cw + i) * 64 + lane] = T[i];
    lds_barrier();
    if (kw > 0) return;
#pragma unroll
    for (int v = 0; v < KS - 1; ++v)
#pragma unroll
      for (int i = 0; i < 2; ++i) T[i] += part[(v * 4 + 2 * cw + i) * 64 + lane];
  }
  if (r16 >= tl.z) return;
  if constexpr (UP) {
    const int he = row_exponent(xm, a.hidden, bound);
    const float sc = ldexpf(1.0f, -he);
    const uint32_t lo = f2h2(sc * swiglu(T[0][0], T[1][0]), sc * swiglu(T[0][1], T[1][1]));
    const uint32_t hi = f2h2(sc * swiglu(T[0][2], T[1][2]), sc * swiglu(T[0][3], T[1][3]));
    if (cb == 0 && cw == 0 && c4 == 0) s.hexp[tl.y + r16] = he;
    *reinterpret_cast<u32x2*>(s.h + (int64_t)(tl.y + r16) * a.inner + 32 * cb + 16 * cw + 4 * c4) =
        (u32x2){lo, hi};
  } else {
    float* const o = s.rows + (int64_t)en * a.hidden + 64 * cb + 32 * cw + 4 * c4;
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<f32x4*>(o + 16 * i) = scaled(wt * T[i], hexp);
  }
}

// ---- tiles of many rows ----

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool H = false>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (H)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// moe_tile_kernel for experts with many rows: a tile of 64 rows against 256
// columns, four waves in a row, each with all rows and 64 columns (two fragments
// of 32), on 32 x 32 x 16 products. x is the A operand: lane (r32, c2) supplies
// row r32 and ends with column r32, rows 8 (e / 4) + 4 c2 + e % 4 of a product's
// 16 sums. An unpacked weight serves two products and a row read from LDS two.
// The k order inside a stage is the packing's: of a fragment's four dwords d and
// the lane groups c = 2 sg + c2 of the two loads sg, product (d, sg) takes the
// 8-column chunks 4 d + 2 sg + c2 of x.
// The rows are copied one stage ahead (two slots), the weights go to registers
// half a stage ahead, once the last of the stage before are unpacked.
// Bound by the vector instructions beside the products: a product of 32 cycles comes
// with 9 of 4 cycles, 4 of them the scaling and 3.5 the unpacking, whose issue it
// blocks for 12, and the card takes its clock back to 2.0 GHz. 16,384 tokens of 9
// columns, hidden 2048, inner 512, 257 experts: up 734 to 747 us, 828 to 843 TFLOP/s.
// In copies without a part, where it took 713: without the row copies 565, the weights
// 607, the offsets 635, the unpacking 663; without any of them 350. Half the unpacking
// with 128 rows a wave and half the columns (twice the row copies) took 760; three
// slots of rows and weights more than two stages ahead, 690 to 700 in 256 registers,
// was not kept.
template <bool UP>
__global__ __launch_bounds__(256)
    __attribute__((amdgpu_waves_per_eu(2, 2))) void
    moe_wide_kernel(MoeArgs a, MoeSpace s) {
  constexpr int MT = 64, XROW = kStageK * 2, XJ = 4, RB = 2;
  __shared__ __align__(16) uint8_t xl0[MT * XROW], xl1[MT * XROW];
  __shared__ int2 row_of[MT];   // a row's token and entry
  __shared__ __align__(16) float wt_of[MT];  // !UP: its weight
  // 2^-exponent of its row of h (UP), or 2^exponent
  __shared__ __align__(16) float hs_of[MT];
  const int K = UP ? a.hidden : a.inner, N = UP ? 2 * a.inner : a.hidden;
  const int P = K >> 7, blocks = (N + 255) >> 8;
  const int n = *s.ntiles * blocks, per = (n + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || idx >= n) return;
  const int tile = idx / blocks, cb = idx - tile * blocks;
  int4 tl = s.tiles[tile];
  tl.x = __builtin_amdgcn_readfirstlane(tl.x);
  tl.y = __builtin_amdgcn_readfirstlane(tl.y);
  tl.z = __builtin_amdgcn_readfirstlane(tl.z);
  if (tl.z == 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, c2 = lane >> 5;
  const bool live = 256 * cb + 64 * wave < N;  // an odd last half block leaves two waves idle

  float bound[2];
  if constexpr (UP)
    for (int i = 0; i < 2; ++i) bound[i] = a.bound[i * a.experts + tl.x];
  RowMax xm;
  if (tid < MT) {
    const int2 pe = s.perm[tl.y + min(tid, tl.z - 1)];
    row_of[tid] = pe;
    if constexpr (UP) {
      xm = load_row_max(s.xmax, pe.x);
    } else {
      wt_of[tid] = a.weights[pe.y];
      hs_of[tid] = ldexpf(1.0f, s.hexp[tl.y + min(tid, tl.z - 1)]);
    }
  }
  // the wave's first 16-row fragment, and the lane's of its 32-column fragment i
  const int64_t f0 = (int64_t)tl.x * (N >> 4) + 16 * cb + (live ? 4 * wave : 0);
  const u32x4* const wp = static_cast<const u32x4*>(UP ? a.w1 : a.w2) + f0 * P * 64;
  const uint32_t* const sb = (UP ? a.sb1 : a.sb2) + f0 * P * 32;
  int fr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) fr[i] = (UP ? i : 2 * i) + (r32 >> 4) * (UP ? 2 : 1);
  const uint16_t* const xbase = UP ? a.x : s.h + (int64_t)tl.y * a.inner;
  __syncthreads();
  uint32_t xvo[XJ];
#pragma unroll
  for (int j = 0; j < XJ; ++j) {
    const int r = 4 * (wave + 4 * j) + (lane >> 4);
    const int64_t at = UP ? (int64_t)row_of[r].x * a.xs : (int64_t)min(r, tl.z - 1) * a.inner;
    xvo[j] = (uint32_t)(at * 2) + 16 * ((lane & 15) ^ (r & 15));
  }
  const int wvo = (fr[0] * P * 64 + 16 * c2 + (r32 & 15)) * 16;
  const int svo = fr[0] * P * 128 + (r32 & 15) * 4, fi = UP ? P : 2 * P;
  auto batch_x = [&](int p, auto slot) {
    constexpr int S = decltype(slot)::value;
    const int in = __builtin_amdgcn_readfirstlane(p < P ? -1 : 0);
    const __amdgpu_buffer_rsrc_t xrs =
        __builtin_amdgcn_make_buffer_rsrc((void*)xbase, (short)0, in, 0x00020000);
#pragma unroll
    for (int j = 0; j < XJ; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xrs,
          (void __attribute__((address_space(3)))*)((S ? xl1 : xl0) + 4 * (wave + 4 * j) * XROW), 16,
          (int)xvo[j], p * XROW, 0, 0);
  };
  u32x4 wr[2][2];
  uint32_t sr[2];
  constexpr int LW = 6;  // loads of a stage's weights
  auto batch_w = [&](int p) {
    const int in = __builtin_amdgcn_readfirstlane(p < P ? -1 : 0);
    const __amdgpu_buffer_rsrc_t wrs =
        __builtin_amdgcn_make_buffer_rsrc((void*)wp, (short)0, in & (4 * P * 1024), 0x00020000);
    const __amdgpu_buffer_rsrc_t srs =
        __builtin_amdgcn_make_buffer_rsrc((void*)sb, (short)0, in & (4 * P * 128), 0x00020000);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
        wr[i][g] = __builtin_amdgcn_raw_buffer_load_b128(wrs, wvo + 512 * g, (p + i * fi) * 1024, 0);
      sr[i] = __builtin_amdgcn_raw_buffer_load_b32(srs, svo, (p + i * fi) * 128, 0);
    }
  };
  uint32_t nib = 0x000F000Fu;
  asm volatile("" : "+v"(nib));
  f32x16 T[2][RB];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int u = 0; u < RB; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) T[i][u][e] = 0.f;

  // the wait counts loads: every copy of rows goes out before the first of the weights
  batch_x(0, std::integral_constant<int, 0>{});
  __builtin_amdgcn_sched_barrier(0);
  batch_w(0);
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (UP)  // beside the first stage's loads
    if (tid < MT) {
      const int he = row_exponent(xm, a.hidden, bound);
      hs_of[tid] = ldexpf(1.0f, -he);
      if (cb == 0 && tid < tl.z) s.hexp[tl.y + tid] = he;
    }
  wait_vm<LW>();
  wait_lgkm0();
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "global");

  // The loop over the stages with the tile's first NB row blocks. A task is a
  // group of 64 k on a row block: 8 products into one of two sets of sums, beside
  // which the task before's sums are scaled into T and the next task's rows are
  // read.
  auto stages = [&](auto nbc) {
    constexpr int NB = decltype(nbc)::value;
    f32x16 y[2][2];
    float sp[2] = {0.f, 0.f};  // scales of the sums not yet in T
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) y[1][i][e] = 0.f;
    u32x4 X[2][2][2], W[2][2][2];
    // byte of chunk c2 of row r32 in a slot; chunk c2 + even number: its bits flipped
    int xrd = r32 * XROW + ((c2 ^ (r32 & 15)) << 4);
    auto rows = [&](const uint8_t* cur, auto tc) {
      constexpr int t = decltype(tc)::value, gl = t / NB, u = t % NB;
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int g = 0; g < 2; ++g)
          X[t & 1][d][g] = *reinterpret_cast<const u32x4*>(
              cur + u * 32 * XROW + (xrd ^ ((8 * gl + 4 * d + 2 * g) << 4)));
    };
    auto unpack = [&](int gl) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
          for (int g = 0; g < 2; ++g) W[i][d][g] = unpack_w<!UP>(wr[i][g][2 * gl + d], nib);
    };
    auto task = [&](const uint8_t* cur, auto tc) {
      constexpr int t = decltype(tc)::value, up = (t + NB - 1) % NB;
      if constexpr (t + 1 < 2 * NB) rows(cur, std::integral_constant<int, t + 1>{});
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) y[t & 1][i][e] = 0.f;
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            y[t & 1][i] = mfma32<!UP>(X[t & 1][d][g], W[i][d][g], y[t & 1][i]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          T[i][up][e] = fmaf(sp[i], y[1 - (t & 1)][i][e], T[i][up][e]);
      if constexpr (t + 1 < 2 * NB) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto step = [&](int p, auto slot, auto lastc) {
      constexpr int S = decltype(slot)::value;
      constexpr bool last = decltype(lastc)::value;
      const uint8_t* const cur = S ? xl1 : xl0;
      asm volatile("" : "+v"(xrd));  // one address register, not one a chunk
      rows(cur, std::integral_constant<int, 0>{});
      if constexpr (!last) batch_x(p + 1, std::integral_constant<int, 1 - S>{});
      unpack(0);
      float s0[2], s1[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s0[i] = bf_lo(sr[i]);
        s1[i] = bf_hi(sr[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
      task(cur, std::integral_constant<int, 0>{});
      sp[0] = s0[0], sp[1] = s0[1];
      if constexpr (NB > 1) task(cur, std::integral_constant<int, 1 % (2 * NB)>{});
      unpack(1);
      if constexpr (!last) batch_w(p + 1);
      __builtin_amdgcn_sched_barrier(0);
      task(cur, std::integral_constant<int, NB>{});
      sp[0] = s1[0], sp[1] = s1[1];
      if constexpr (NB > 1) task(cur, std::integral_constant<int, NB + 1 < 2 * NB ? NB + 1 : NB>{});
      if constexpr (!last) {
        wait_vm<LW>();  // the rows; the weights are waited for where they are unpacked
        wait_lgkm0();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "global");
      }
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    int p = 0;
#pragma nounroll
    for (; p + 2 <= P; p += 2) {
      step(p, S0{}, std::false_type{});
      step(p + 1, S1{}, std::false_type{});
    }
    if (p < P) step(p, S0{}, std::true_type{});
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) T[i][NB - 1][e] = fmaf(sp[i], y[1][i][e], T[i][NB - 1][e]);
  };
  const int nb = (tl.z + 31) >> 5;
  if (nb == 2)
    stages(std::integral_constant<int, 2>{});
  else
    stages(std::integral_constant<int, 1>{});

  // The offsets' sum: both lane groups hold the same octet of X, one against b and
  // the other against -offset s.
  const int gp = gpad(K), go = gp >> 3;
  const float f = c2 ? UP ? -kOffsetX : -kOffsetH : 1.0f;
#pragma nounroll
  for (int o = 0; o < go; ++o) {
    u32x4 B[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int ps = 4 * o + q;
        const uint32_t v = ps < P ? sb[(fr[i] * P + ps) * 32 + (c2 ? 0 : 16) + (r32 & 15)] : 0u;
        B[i][q] = f2bf2(f * bf_lo(v), f * bf_hi(v));
      }
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      if (32 * u >= tl.z) continue;
      const int r = min(u * 32 + r32, tl.z - 1);
      const uint16_t* const xg =
          UP ? s.xs + (int64_t)row_of[r].x * 3 * gp : s.hs + (int64_t)(tl.y + r) * 3 * gp;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const u32x4 xp = *reinterpret_cast<const u32x4*>(xg + k * gp + 8 * o);
#pragma unroll
        for (int i = 0; i < 2; ++i) T[i][u] = mfma32(xp, B[i], T[i][u]);
      }
    }
  }

  if constexpr (UP) {
    // h goes through LDS, so that rows are written 16 bytes a lane; the slots are
    // free once every wave is here.
    lds_barrier();
    uint16_t* const hb = reinterpret_cast<uint16_t*>(xl0);  // [MT][128], chunks of 8 swizzled
    const int c = 32 * wave + r32;
#pragma unroll
    for (int u = 0; u < RB; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r0 = 32 * u + 8 * q + 4 * c2;
        const f32x4 sc = *reinterpret_cast<const f32x4*>(&hs_of[r0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + e;
          if (live)
            hb[r * 128 + 8 * ((c >> 3) ^ (r & 15)) + (c & 7)] = __builtin_bit_cast(
                uint16_t, (_Float16)(sc[e] * swiglu(T[0][u][4 * q + e], T[1][u][4 * q + e])));
        }
      }
    lds_barrier();
    const int gi = gpad(a.inner), ch = tid & 15, cols = min(128, a.inner - 128 * cb);
#pragma unroll
    for (int j = 0; j < MT / 16; ++j) {
      const int r = 16 * j + (tid >> 4);
      if (r >= tl.z || 8 * ch >= cols) continue;
      const u32x4 v = *reinterpret_cast<const u32x4*>(hb + r * 128 + 8 * (ch ^ (r & 15)));
      *reinterpret_cast<u32x4*>(s.h + (int64_t)(tl.y + r) * a.inner + 128 * cb + 8 * ch) = v;
      float t = 0.f;
      uint32_t m = 0;  // |h| as the order of its bits
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        t += h_lo(v[q]) + h_hi(v[q]);
        m = max(m, max_abs2(v[q]));
      }
      t = sum8(t);
      m = max8(m);
      if ((ch & 7) == 0) {
        uint16_t* const dst = s.hs + (int64_t)(tl.y + r) * 3 * gi;
        store_split(t, dst + 2 * cb + (ch >> 3), gi);
        if (a.inner <= kWideInner) s.hmax[(tl.y + r) * 8 + 2 * cb + (ch >> 3)] = (uint16_t)m;
        if (cb == blocks - 1 && ch == 0)  // the padded groups
          for (int g = a.inner >> 6; g < gi; ++g) store_split(0.f, dst + g, gi);
      }
    }
  } else {
    if (!live) return;
    // a store writes 32 columns, 128 bytes, of two rows
    float* const rows = s.rows + 256 * cb + 64 * wave + r32;
#pragma unroll
    for (int u = 0; u < RB; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r0 = 32 * u + 8 * q + 4 * c2;
        const f32x4 wt = *reinterpret_cast<const f32x4*>(&wt_of[r0]);
        const f32x4 hs = *reinterpret_cast<const f32x4*>(&hs_of[r0]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r0 + e < tl.z) {
            float* const o = rows + (int64_t)row_of[r0 + e].y * a.hidden;
            o[0] = wt[e] * T[0][u][4 * q + e] * hs[e];
            o[32] = wt[e] * T[1][u][4 * q + e] * hs[e];
          }
      }
  }
}

// Down for experts with many rows and inner up to 512: a tile of 64 rows stays in
// LDS (four stages) while the work-group takes `run` blocks of 256 columns one
// after the other, weights ahead across blocks; no wave waits for another.
// Products, tasks and roles as in moe_wide_kernel, and so is its bound.
// A row goes out in f16 under an exponent of its own: |down h| is at most the largest
// sum of |w| over a column's inputs times the largest |h|, and the power of two above
// that and the weight is brought to 2^15. A value keeps 11 bits down to 2^-29 of the
// bound and 2^-40 of it absolutely; only the result's own 8 bits follow. The same
// 16,384 tokens: 415 us, 745 TFLOP/s, and 102 for their sum. In f32 it was 460 and 215.
// In bf16, at 410 and 101, the rows' rounding moved the result by as much as its own
// does, 0.0017 of its norm; so it stays at the 0.0017.
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void
    moe_wide_down_kernel(MoeArgs a, MoeSpace s, int run) {
  constexpr int MT = 64, XROW = kStageK * 2, SLOT = MT * XROW;
  __shared__ __align__(16) uint8_t xl[4 * SLOT];
  __shared__ __align__(16) uint16_t stage_out[4][16 * 64];
  __shared__ u32x4 sums[MT][3];  // a row's split group sums: hi, mid, lo octet
  __shared__ int en_of[MT];
  __shared__ __align__(16) float wt_of[MT];  // weights times 2^-exponent
  const int P = a.inner >> 7, N = a.hidden, blocks = (N + 255) >> 8;
  const int chunks = (blocks + run - 1) / run;
  const int n = *s.ntiles * chunks, per = (n + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || idx >= n) return;
  const int tile = idx / chunks;
  const int cb0 = (idx - tile * chunks) * run, cb1 = min(cb0 + run, blocks);
  int4 tl = s.tiles[tile];
  tl.x = __builtin_amdgcn_readfirstlane(tl.x);
  tl.y = __builtin_amdgcn_readfirstlane(tl.y);
  tl.z = __builtin_amdgcn_readfirstlane(tl.z);
  if (tl.z == 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, c2 = lane >> 5;

  const int bound = __builtin_amdgcn_readfirstlane(
      __builtin_amdgcn_frexp_expf(a.bound[2 * a.experts + tl.x]));
  // the rows of all stages, and what goes with a row
  {
    const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(s.h + (int64_t)tl.y * a.inner), (short)0, -1, 0x00020000);
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * (wave + 4 * j) + (lane >> 4);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            xrs,
            (void __attribute__((address_space(3)))*)(xl + p * SLOT + 4 * (wave + 4 * j) * XROW), 16,
            min(r, tl.z - 1) * a.inner * 2 + 16 * ((lane & 15) ^ (r & 15)), p * XROW, 0, 0);
      }
    if (tid < 3 * MT)
      sums[tid / 3][tid % 3] = *reinterpret_cast<const u32x4*>(
          s.hs + ((int64_t)tl.y + min(tid / 3, tl.z - 1)) * 24 + 8 * (tid % 3));
    if (tid < MT) {
      const int en = s.perm[tl.y + min(tid, tl.z - 1)].y;
      const float w = a.weights[en];
      const u32x4 hm =
          *reinterpret_cast<const u32x4*>(s.hmax + (tl.y + min(tid, tl.z - 1)) * 8);
      uint32_t m = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q)  // stages: two groups each
        if (q < P) m = max(m, max(hm[q] & 0xFFFFu, hm[q] >> 16));
      // 2^b is above the row's values before the weight and h's own power of two, 2^(b +
      // exponent of w) after the weight
      const int b = __builtin_amdgcn_frexp_expf(h_lo(m)) + bound;
      const int e = max(-100, min(b, 128)) + __builtin_amdgcn_frexp_expf(w) - 15;
      en_of[tid] = en;
      wt_of[tid] = ldexpf(w, -e);
      if (cb0 == 0 && tid < tl.z) s.exps[en] = e + s.hexp[tl.y + tid];
    }
    wait_vm<0>();
    __syncthreads();
  }
  const int f16 = r32 >> 4;  // which of a column fragment's two 16-row fragments
  const u32x4* const wp = static_cast<const u32x4*>(a.w2) + (int64_t)tl.x * (N >> 4) * P * 64;
  const uint32_t* const sb = a.sb2 + (int64_t)tl.x * (N >> 4) * P * 32;
  const int wvo = (f16 * P * 64 + 16 * c2 + (r32 & 15)) * 16;
  const int svo = f16 * P * 128 + (r32 & 15) * 4;
  // this wave's blocks: those whose 64 columns are there
  const int cbw = min(cb1, (N - 64 * wave + 255) >> 8);
  if (cb0 >= cbw) return;
  u32x4 wr[2][2];
  uint32_t sr[2], ob[2][4];
  auto batch_w = [&](int cb, int p) {
    const int in = __builtin_amdgcn_readfirstlane(cb < cbw ? -1 : 0);
    const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)wp, (short)0, in & ((N >> 4) * P * 1024), 0x00020000);
    const __amdgpu_buffer_rsrc_t srs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)sb, (short)0, in & ((N >> 4) * P * 128), 0x00020000);
    const int f0 = 16 * cb + 4 * wave;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
        wr[i][g] = __builtin_amdgcn_raw_buffer_load_b128(wrs, wvo + 512 * g,
                                                         ((f0 + 2 * i) * P + p) * 1024, 0);
      sr[i] = __builtin_amdgcn_raw_buffer_load_b32(srs, svo, ((f0 + 2 * i) * P + p) * 128, 0);
    }
  };
  uint32_t nib = 0x000F000Fu;
  asm volatile("" : "+v"(nib));

  auto body = [&](auto nbc) {
    constexpr int NB = decltype(nbc)::value;
    f32x16 T[2][NB], y[2][2];
    float sp[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        y[1][i][e] = 0.f;
#pragma unroll
        for (int u = 0; u < NB; ++u) T[i][u][e] = 0.f;
      }
    u32x4 X[2][2][2], W[2][2][2];
    const int xrd = r32 * XROW + ((c2 ^ (r32 & 15)) << 4);
    auto rows = [&](int at, auto tc) {
      constexpr int t = decltype(tc)::value, gl = t / NB, u = t % NB;
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int g = 0; g < 2; ++g)
          X[t & 1][d][g] = *reinterpret_cast<const u32x4*>(
              xl + u * 32 * XROW + (at ^ ((8 * gl + 4 * d + 2 * g) << 4)));
    };
    auto unpack = [&](int gl) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
          for (int g = 0; g < 2; ++g) W[i][d][g] = unpack_w<true>(wr[i][g][2 * gl + d], nib);
    };
    auto task = [&](int at, auto tc) {
      constexpr int t = decltype(tc)::value, up = (t + NB - 1) % NB;
      if constexpr (t + 1 < 2 * NB) rows(at, std::integral_constant<int, t + 1>{});
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) y[t & 1][i][e] = 0.f;
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            y[t & 1][i] = mfma32<true>(X[t & 1][d][g], W[i][d][g], y[t & 1][i]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          T[i][up][e] = fmaf(sp[i], y[1 - (t & 1)][i][e], T[i][up][e]);
      if constexpr (t + 1 < 2 * NB) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    batch_w(cb0, 0);
    for (int cb = cb0; cb < cbw; ++cb) {
#pragma nounroll
      for (int p = 0; p < P; ++p) {
        int at = xrd + p * SLOT;
        asm volatile("" : "+v"(at));
        rows(at, std::integral_constant<int, 0>{});
        unpack(0);
        const float s0[2] = {bf_lo(sr[0]), bf_lo(sr[1])}, s1[2] = {bf_hi(sr[0]), bf_hi(sr[1])};
        __builtin_amdgcn_sched_barrier(0);
        task(at, std::integral_constant<int, 0>{});
        sp[0] = s0[0], sp[1] = s0[1];
        if constexpr (NB > 1) task(at, std::integral_constant<int, 1 % (2 * NB)>{});
        unpack(1);
        // the sums so far are not moved behind the branch
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int u = 0; u < NB; ++u) asm volatile("" : "+v"(T[i][u]));
        if (p + 1 < P) {
          batch_w(cb, p + 1);
        } else {
          batch_w(cb + 1, 0);
          // biases (lanes c2 = 0) or scales (c2 = 1) of the block's stages
          const __amdgpu_buffer_rsrc_t srs = __builtin_amdgcn_make_buffer_rsrc(
              (void*)sb, (short)0, (N >> 4) * P * 128, 0x00020000);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              ob[i][q] = __builtin_amdgcn_raw_buffer_load_b32(
                  srs, svo + (c2 ? 0 : 64), ((16 * cb + 4 * wave + 2 * i) * P + min(q, P - 1)) * 128, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        task(at, std::integral_constant<int, NB>{});
        sp[0] = s1[0], sp[1] = s1[1];
        if constexpr (NB > 1) task(at, std::integral_constant<int, NB + 1 < 2 * NB ? NB + 1 : NB>{});
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) T[i][NB - 1][e] = fmaf(sp[i], y[1][i][e], T[i][NB - 1][e]);
        sp[i] = 0.f;
      }
      // the offsets' sum: both lane groups hold the same octet of X, against b
      // and against -offset s
      u32x4 B[2];
      const float f = c2 ? -kOffsetH : 1.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          B[i][q] = q < P ? f2bf2(f * bf_lo(ob[i][q]), f * bf_hi(ob[i][q])) : 0u;
#pragma unroll
      for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          const u32x4 xp = sums[32 * u + r32][k];
#pragma unroll
          for (int i = 0; i < 2; ++i) T[i][u] = mfma32(xp, B[i], T[i][u]);
        }
      // Through LDS, 16 rows at a time, so that rows are written 16 bytes a lane:
      // 8-column chunk ch of row r at chunk ch ^ (r % 8). The lane's first byte is
      // that of row 4 c2, column r32; other rows and columns flip or add bits.
      char* const so = reinterpret_cast<char*>(stage_out[wave]);
      int wat = 512 * c2 + (((r32 >> 3) | 4 * c2) << 4) + 2 * (r32 & 7);
      int rat = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
      asm volatile("" : "+v"(wat), "+v"(rat));  // addresses formed here, not kept
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int r0 = 32 * u + 16 * hf;
          if (r0 >= tl.z) break;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const v4f wt = *reinterpret_cast<const v4f*>(&wt_of[r0 + 8 * g + 4 * c2]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                *reinterpret_cast<_Float16*>(so + (wat ^ ((e << 4) | (i << 6))) + 128 * e + 1024 * g) =
                    (_Float16)(wt[e] * T[i][u][8 * hf + 4 * g + e]);
          }
          wait_lgkm0();
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = r0 + 8 * j + (lane >> 3);
            const u32x4 v = *reinterpret_cast<const u32x4*>(so + rat + 1024 * j);
            if (r < tl.z)
              *reinterpret_cast<u32x4*>(reinterpret_cast<_Float16*>(s.rows) + (int64_t)en_of[r] * N +
                                        256 * cb + 64 * wave + 8 * (lane & 7)) = v;
          }
          wait_lgkm0();
          __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) T[i][u][e] = 0.f;
    }
  };
  if (tl.z > 32)
    body(std::integral_constant<int, 2>{});
  else
    body(std::integral_constant<int, 1>{});
}

// out[t] = the sum of its entries' rows in column order. A thread per 4 columns, B
// rows' loads at a time; rows of ids outside the layer are read as they are in the
// work-space and left out. Bound by reading the rows, in small calls by latency:
// those take all of a token's rows at once, in small work-groups over more CUs.
template <int B>
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs a, const float* rows) {
  const int q = a.hidden / 4;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)a.T * q) return;
  const int64_t t = i / q;
  const int c = (int)(i - t * q);
  const f32x4* const r = reinterpret_cast<const f32x4*>(rows) + t * a.k * q + c;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < a.k; j0 += B) {
    f32x4 v[B];
    bool in[B];
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (j0 + j < a.k) {
        v[j] = __builtin_nontemporal_load(r + (int64_t)(j0 + j) * q);
        in[j] = (uint32_t)a.ids[t * a.k + j0 + j] < (uint32_t)a.experts;
      }
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (j0 + j < a.k && in[j]) y += v[j];
  }
  *reinterpret_cast<u32x2*>(a.out + t * a.os + c * 4) =
      (u32x2){f2bf2(y[0], y[1]), f2bf2(y[2], y[3])};
}

// The same of f16 rows: a thread per 8 columns.
__global__ __launch_bounds__(256) void moe_combine_half_kernel(MoeArgs a, MoeSpace s) {
  constexpr int B = 4;
  const int q = a.hidden / 8;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)a.T * q) return;
  const int64_t t = i / q;
  const int c = (int)(i - t * q);
  const f16x8* const r = reinterpret_cast<const f16x8*>(s.rows) + t * a.k * q + c;
  float y[8] = {};
  for (int j0 = 0; j0 < a.k; j0 += B) {
    f16x8 v[B];
    int e[B];
    bool in[B];
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (j0 + j < a.k) {
        v[j] = __builtin_nontemporal_load(r + (int64_t)(j0 + j) * q);
        e[j] = s.exps[t * a.k + j0 + j];
        in[j] = (uint32_t)a.ids[t * a.k + j0 + j] < (uint32_t)a.experts;
      }
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (j0 + j < a.k && in[j])
#pragma unroll
        for (int n = 0; n < 8; ++n) y[n] += ldexpf((float)v[j][n], e[j]);
  }
  u32x2* const o = reinterpret_cast<u32x2*>(a.out + t * a.os + c * 8);
  o[0] = (u32x2){f2bf2(y[0], y[1]), f2bf2(y[2], y[3])};
  o[1] = (u32x2){f2bf2(y[4], y[5]), f2bf2(y[6], y[7])};
}

// ---- launches ----

template <typename... Par, typename... Arg>
hipError_t launch(void (*kernel)(Par...), int64_t groups, int threads, size_t lds, hipStream_t stream,
                  Arg... args) {
  hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(threads), lds, stream, args...);
  return hipGetLastError();
}

#define MOE_TRY(x)                        \
  do {                                    \
    const hipError_t e_ = (x);            \
    if (e_ != hipSuccess) return e_;      \
  } while (0)

// Work-groups of `blocks` per tile slot, the same number for every XCD.
int64_t tile_groups(int64_t slots, int blocks) { return (slots * blocks + 7) & ~(int64_t)7; }

// Two parts of the stages where a wave would have 8 or more: 8 tokens at hidden
// 2048, inner 512, 257 experts, 9 columns, up 16.4 us against 22.9 and 20.4 in four
// parts, 64 tokens 44.1 / 44.9 / 53.5; down, of 4 stages, 10.6 in one part and 12.7 in
// two at 8 tokens, 27.8 / 32.5 at 64.
template <bool UP>
hipError_t launch_stream(const MoeArgs& a, const MoeSpace& s, int64_t slots) {
  const int64_t groups = tile_groups(slots, UP ? a.inner / 32 : a.hidden / 64);
  if ((UP ? a.hidden : a.inner) >= 8 * kStageK)
    return launch(moe_stream_kernel<2, UP>, groups, 256, 0, a.stream, a, s);
  return launch(moe_stream_kernel<1, UP>, groups, 128, 0, a.stream, a, s);
}

template <int MW>
hipError_t launch_tiles(const MoeArgs& a, const MoeSpace& s, int64_t slots) {
  MOE_TRY(launch(moe_tile_kernel<MW, true>, tile_groups(slots, a.inner / 64), 256, 0, a.stream, a, s));
  return launch(moe_tile_kernel<MW, false>, tile_groups(slots, a.hidden / 128), 256, 0, a.stream, a,
                s);
}

hipError_t launch_wide(const MoeArgs& a, const MoeSpace& s, int64_t slots, int64_t tiles) {
  MOE_TRY(launch(moe_wide_kernel<true>, tile_groups(slots, a.inner / 128), 256, 0, a.stream, a, s));
  const int blocks = (a.hidden + 255) / 256;
  if (a.inner > kWideInner)
    return launch(moe_wide_kernel<false>, tile_groups(slots, blocks), 256, 0, a.stream, a, s);
  // Long runs, as long as they leave three work-groups for each of the 512 that run
  // side by side. The whole call in runs of 8 / 4 / 2 / 1 blocks: 16,384 tokens (2,400
  // tiles) 1197 / 1208 / 1221 / 1259 us, 4,000 (690) 379 / 368 / 364 / 374.
  int run = blocks;
  while (run > 1 && tiles * ((blocks + run - 1) / run) < 1536) run = (run + 1) / 2;
  return launch(moe_wide_down_kernel, tile_groups(slots, (blocks + run - 1) / run), 256, 0, a.stream,
                a, s, run);
}

}  // namespace

hipError_t launch_moe_pack(const MoePackArgs& a) {
  const int blocks = (a.n * (a.k / 128) * 4 + 255) / 256;
  hipLaunchKernelGGL(moe_pack_kernel, dim3(blocks < 64 ? blocks : 64, a.experts), dim3(256), 0,
                     a.stream, a);
  return hipGetLastError();
}

hipError_t launch_moe_bound(const MoePackArgs& a, bool down, float* bound) {
  hipLaunchKernelGGL(moe_bound_kernel, dim3((a.n + 63) / 64, a.experts), dim3(256), 0, a.stream, a,
                     down ? kOffsetH : kOffsetX, bound);
  return hipGetLastError();
}

// A pass's rows of x are reached by 32-bit byte offsets.
int moe_pass_tokens(int k, int64_t x_stride) {
  const int64_t n = kPassEntries / k, reach = kReach / 2 / x_stride;
  return (int)(n < reach ? n : reach > 1 ? reach : 1);
}

size_t moe_workspace_bytes(int hidden, int inner, int experts, int T, int k) {
  int64_t entries = (int64_t)T * k, tokens = T;
  if (entries > kPassEntries) entries = kPassEntries;
  if (tokens > kPassEntries) tokens = kPassEntries;
  return moe_space(nullptr, hidden, inner, experts, tokens, entries).bytes;
}

hipError_t launch_moe(const MoeArgs& a) {
  const int entries = a.T * a.k;
  MoeSpace s = moe_space(a.workspace, a.hidden, a.inner, a.experts, a.T, entries);
  if (entries <= kFewEntries && a.T <= kFewTokens) {
    MOE_TRY(launch(moe_few_up_kernel, entries * (a.inner / 16), 256, 0, a.stream, a, s.h));
    return launch(moe_few_down_kernel, a.T * (a.hidden / 16), 64 * (a.k < 16 ? a.k : 16), 0, a.stream,
                  a, s.h);
  }
  // The kernel by the rows that an expert has on average. At hidden 2048, inner
  // 512, 257 experts, 9 columns, tiles of 16 rows by the stream kernel / 16 / 32 /
  // 64 rows: 64 tokens (mean 2) 77 / 85 / 89 / 108 us, 200 (7) 101 / 104 / 110 / 132,
  // 317 (11) 121 / 113 / 119 / 137, 600 (21) 169 / 145 / 138 / 147, 1000 (35) 244 / 194 /
  // 178 / 167, 2000 (70) 428 / 329 / 281 / 226. Tiles of 64 rows also want a work-group
  // for most of the 512 that run side by side (hidden 1024, inner 1408, 32 experts, 4
  // columns: 1000 tokens, 312 work-groups, 78 us by 32 rows and 77 by 64; 1500 tokens,
  // 436, 104 / 91).
  const int mean = entries / a.experts;
  const int64_t wide_tiles = max_tiles(entries, a.experts, 64) - a.experts / 2;
  const bool wide = entries >= wide_entries(a.hidden, a.experts);
  const bool stream = mean < 8;
  const int rows = wide ? 64 : mean <= 16 ? 16 : 32;
  const int64_t slots = max_tiles(entries, a.experts, rows);
  const int64_t sum_groups = ((int64_t)a.T * 8 * gpad(a.hidden) + kPlanThreads - 1) / kPlanThreads;
  if (stream) s.xs = nullptr;  // the maxima only
  if (entries <= kPlanEntries) {
    MOE_TRY(launch(moe_plan_kernel, a.experts + sum_groups, kPlanThreads, 0, a.stream, a, rows, s));
  } else {
    const int chunks = (entries + kChunk - 1) / kChunk;
    MOE_TRY(launch(moe_count_kernel, chunks + sum_groups, kPlanThreads, a.experts * 4, a.stream, a,
                   chunks, s));
    MOE_TRY(launch(moe_place_kernel, chunks, kPlanThreads, a.experts * 8, a.stream, a, rows, s));
  }
  if (wide) {
    MOE_TRY(launch_wide(a, s, slots, wide_tiles));
  } else if (stream) {
    MOE_TRY(launch_stream<true>(a, s, slots));
    MOE_TRY(launch_stream<false>(a, s, slots));
  } else {
    MOE_TRY(rows == 16 ? launch_tiles<1>(a, s, slots) : launch_tiles<2>(a, s, slots));
  }
  const int64_t n = (int64_t)a.T * (a.hidden / 4);
  if (wide && a.inner <= kWideInner)
    return launch(moe_combine_half_kernel, (n / 2 + 255) / 256, 256, 0, a.stream, a, s);
  if (n < 1 << 17) return launch(moe_combine_kernel<16>, (n + 63) / 64, 64, 0, a.stream, a, s.rows);
  return launch(moe_combine_kernel<4>, (n + 255) / 256, 256, 0, a.stream, a, s.rows);
}

}  // namespace gdn
