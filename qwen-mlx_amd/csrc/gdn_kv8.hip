// gdn_kv8.hip -- the 8-bit paged KV cache: tables and maps of a step from request
// lengths, new tokens into pages, and pages read back.
//
// Page layout, one layer: [2 (K, V)][Hkv][64 * D] e4m3 bytes, every 64 * D tile in the
// order that attention's MFMA operands are loaded, so that a wave's 16-byte loads read
// 1 KiB in one piece:
//   K (key kk, dim d): [kk/16][d/64][(d%64)/16][kk%16][d%16] -- a lane's 16 bytes are 16
//       dims of a key: the A operand (16 keys, 32-deep k = dims) of two products
//   V (key kk, dim d): [kk/32][d/16][(kk/4)%2][d%16][(kk/8)%2][(kk/16)%2][kk%4] -- a lane's 16
//       bytes are 16 keys of a dim, every other four of 32: the A operand of two products (32
//       dims, 16-deep k = keys), keys in the order in which the score accumulators hold them;
//       with its halves exchanged between the wave's halves, of two of 16 dims, 32 keys deep
// One exponent per page, K or V, and head: exps[page][2][Hkv], in the low 8 bits of a word.
#include "gdn_common.h"

namespace gdn {

namespace {

constexpr int kPage = 64;
constexpr int kEMin = -40, kEMax = 56;
constexpr int kNanFlag = 1 << 16;  // of an exponent word: the tile holds a NaN

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int k_byte(int kk, int d, int D) {
  return ((kk >> 4) * (D >> 6) + (d >> 6)) * 1024 + (((d >> 4) & 3) * 16 + (kk & 15)) * 16 + (d & 15);
}
__device__ __forceinline__ int v_byte(int kk, int d, int D) {
  return (kk >> 5) * 32 * D + (d >> 4) * 512 + (((kk >> 2) & 1) * 16 + (d & 15)) * 16 +
         ((kk >> 3) & 1) * 8 + ((kk >> 4) & 1) * 4 + (kk & 3);
}

// 2^e of a normal f32, e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Value of an e4m3 byte (bit patterns 0x7f and 0xff: NaN).
__device__ __forceinline__ float e4m3_value(uint32_t b) {
  return __builtin_amdgcn_cvt_f32_fp8(b, 0);
}

// Two values, |.| <= 448 or beyond by the exponent's clamp, to e4m3, ties to even;
// infinities and NaN to NaN. The conversion's own behaviour past 448 does not matter.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  const float ca = __builtin_amdgcn_fmed3f(a, -448.f, 448.f);
  const float cb = __builtin_amdgcn_fmed3f(b, -448.f, 448.f);
  uint32_t r = __builtin_amdgcn_cvt_pk_fp8_f32(ca, cb, 0, false) & 0xffffu;
  if (!(fabsf(a) < INFINITY)) r = (r & 0xff00u) | 0x7fu;
  if (!(fabsf(b) < INFINITY)) r = (r & 0x00ffu) | 0x7f00u;
  return r;
}

// The least e in [kEMin, kEMax] with amax <= 448 * 2^e; amax finite, given as f32 bits >= 0.
__device__ __forceinline__ int exponent_of(uint32_t bits) {
  // amax = 1.f * 2^x: 448 = 1.75 * 2^8
  const int x = (int)(bits >> 23) - 127;
  const int e = x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return bits < 0x00800000u ? kEMin : min(max(e, kEMin), kEMax);
}

// Row of item g in the prefix sums pre[0 .. n] (pre[n] > g): the last row whose items start
// at or before g. By the wave, 64 rows at a time. Where the plan has fewer rows than n, an item
// behind theirs falls to the first row behind them, which holds nothing.
__device__ __forceinline__ int row_of(const int32_t* __restrict__ pre, int n, int g) {
  const int lane = threadIdx.x & 63;
  int r = 0;
  for (int b = 0; b < n; b += 64) {
    const int v = b + lane < n ? pre[b + lane + 1] : INT32_MAX;
    const int c = __popcll(__ballot(v <= g));
    r = b + c;
    if (c < 64) break;
  }
  return r;
}

}  // namespace

// ------------------------------------------------------------------- the step --

namespace {

// Sum over the work-group's threads before this one (exclusive), and the total; red holds
// a value per wave and is free again after the next barrier.
template <int TH>
__device__ __forceinline__ int block_scan(int v, int* red, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int u = __shfl_up(s, off, 64);
    s += lane >= off ? u : 0;
  }
  if (lane == 63) red[w] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < TH / 64; ++i) {
    before += i < w ? red[i] : 0;
    total += red[i];
  }
  __syncthreads();
  return before + s - v;
}

// Tokens t of the step, each its row by search in cu (LDS or memory).
__device__ __forceinline__ void map_token(const Kv8Plan& p, const int32_t* cu, int t) {
  int pos = -1, place = -1, row = -2;
  if (t < cu[p.n]) {
    int lo = 0, hi = p.n;  // the row: cu[row] <= t < cu[row + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    const Kv8Row r = p.rows[lo];
    row = -1;
    if (r.fresh > 0) {
      row = lo;
      pos = r.pos + t - r.cu;
      place = p.table[(size_t)r.slot * p.max_pages + pos / kPage] * kPage + pos % kPage;
    }
  }
  p.pos[t] = pos;
  p.map[t] = place;
  p.tok_row[t] = row;
}

// Tokens that the plan's own work-group maps: 6,400 take 11 us, 14 with a kernel for them; 16,000
// take 16, and 14.
constexpr int kMapHere = 8192;

// One work-group: prefix sums over the rows (R consecutive rows a thread), pages given
// back, then pages taken, both in row order. Bound by latency: a load of the rows, four or five
// scans and the tables' round trips, and where pages move a load and a store for each row of a
// wave in turn. 64 rows that move none 4.9 us, a page each 6.8, 16 each 18.6, 65 each 25.6; 700 rows
// that move none 6.2, 4,185 pages 13.3.
template <int TH, int R>
__global__ __launch_bounds__(TH) void kv8_plan_kernel(Kv8Plan p, const int32_t* __restrict__ slots,
                                                      const int32_t* lens,
                                                      const int32_t* __restrict__ ntok,
                                                      int32_t* lens_out) {
  __shared__ int red[TH / 64];
  __shared__ int32_t scu[TH * R + 1];
  __shared__ int taken;
  const int tid = threadIdx.x, lane = tid & 63;
  int slot[R], len[R], fresh[R], cu[R], have[R], need[R];
  bool ok[R];
  uint32_t flags = 0;
  if (tid == 0) taken = 0;
  const int count = *p.free_count, used = p.used[0], used_t = p.used[1];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = tid * R + i;
    slot[i] = r < p.n ? slots[r] : -1;
    len[i] = r < p.n ? lens[r] : 0;
    fresh[i] = r < p.n ? ntok[r] : 0;
    ok[i] = slot[i] >= 0 && slot[i] < p.num_slots;
    if (slot[i] >= p.num_slots) flags |= GDN_FLAG_BAD_SLOT;
    if (ok[i]) atomicMin(p.mark + slot[i], r);
  }
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = tid * R + i;
    have[i] = ok[i] ? p.owned[slot[i]] : 0;
    if (ok[i] && __hip_atomic_load(p.mark + slot[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != r) {
      flags |= GDN_FLAG_DUP_SLOT;
      ok[i] = false;
    }
    if (slot[i] >= 0 && (len[i] < 0 || fresh[i] < 0 || fresh[i] > p.max_row ||
                         (int64_t)len[i] + fresh[i] > (int64_t)p.max_pages * kPage)) {
      flags |= GDN_FLAG_BAD_SEQLENS;
      ok[i] = false;
    }
    // tokens of the packing: a row's own unless it is padding
    fresh[i] = slot[i] >= 0 ? min(max(fresh[i], 0), p.T + 1) : 0;
    cu[i] = sum;
    sum += fresh[i];
  }
  int total;
  const int c0 = block_scan<TH>(sum, red, total);
  if (tid == 0) scu[p.n] = p.cu[p.n] = total;
  int gives = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = tid * R + i;
    cu[i] += c0;
    if (r < p.n) scu[r] = p.cu[r] = cu[i];
    if (ok[i] && cu[i] + fresh[i] > p.T) {
      flags |= GDN_FLAG_BAD_SEQLENS;
      ok[i] = false;
    }
    need[i] = ok[i] ? (len[i] + fresh[i] + kPage - 1) / kPage : have[i];
    gives += max(have[i] - need[i], 0);
  }
  int given;
  int at = count + block_scan<TH>(gives, red, given);
  // A row's moves: `m` pages between table positions t0 + s j and stack places f0 + j.
  // A wave takes rows of many pages together, a thread its short ones alone.
  auto move = [&](int m, int sl, int t0, int ts, int f0, int fs, bool push) {
    auto one = [&](int sl_, int t, int f) {
      int32_t* const e = p.table + (size_t)sl_ * p.max_pages + t;
      if (push) {
        p.free_pages[f] = *e;
        *e = -1;
      } else {
        *e = p.free_pages[f];
        p.free_pages[f] = -1;
      }
    };
    constexpr int kAlone = 4;
    if (m > 0 && m <= kAlone)
      for (int j = 0; j < m; ++j) one(sl, t0 + ts * j, f0 + fs * j);
    uint64_t many = __ballot(m > kAlone);
    while (many) {
      const int l = __ffsll((unsigned long long)many) - 1;
      many &= many - 1;
      const int m_ = __builtin_amdgcn_readlane(m, l), s_ = __builtin_amdgcn_readlane(sl, l);
      const int t_ = __builtin_amdgcn_readlane(t0, l), f_ = __builtin_amdgcn_readlane(f0, l);
      for (int j = lane; j < m_; j += 64) one(s_, t_ + ts * j, f_ + fs * j);
    }
  };
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int m = max(have[i] - need[i], 0);
    move(m, slot[i], have[i] - 1, -1, at, 1, true);
    at += m;
  }
  int grows = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) grows += max(need[i] - have[i], 0);
  int all;
  int before = block_scan<TH>(grows, red, all);  // its barriers also order the stack's writes
  const int avail = count + given;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    int m = max(need[i] - have[i], 0);
    if (m > 0 && before + m > avail) {
      flags |= GDN_FLAG_NO_PAGES;
      ok[i] = false;
    }
    const int b = before;
    before += m;
    if (!ok[i]) m = 0;
    if (m > 0) atomicMax(&taken, before);  // admitted rows come before refused ones
    move(m, slot[i], have[i], 1, avail - 1 - b, -1, false);
  }
  // pages that the row's tokens fall into, attention's tiles
  const int tpt = kKv8TileWaves * (32 / (p.Hq / p.Hkv));
  int touched[R], tiles[R], nblk = 0, ntile = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = tid * R + i;
    const int tok = ok[i] ? fresh[i] : 0;
    touched[i] = tok > 0 ? (len[i] + tok - 1) / kPage - len[i] / kPage + 1 : 0;
    tiles[i] = tok >= kKv8TileTokens ? (tok + tpt - 1) / tpt : 0;
    nblk += touched[i];
    ntile += tiles[i];
    if (r >= p.n) continue;
    p.rows[r] = Kv8Row{ok[i] ? slot[i] : -1, len[i], tok, cu[i]};
    if (ok[i]) p.owned[slot[i]] = need[i];
    if (lens_out) lens_out[r] = ok[i] ? len[i] + tok : len[i];
    if (slot[i] >= 0 && slot[i] < p.num_slots) p.mark[slot[i]] = INT32_MAX;
  }
  int none;
  int t1 = p.max_row >= kKv8TileTokens ? block_scan<TH>(ntile, red, none) : 0;
  int b0 = block_scan<TH>(nblk, red, total);  // and orders the tables for the tokens
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = tid * R + i;
    if (r >= p.n) continue;
    p.blocks[r] = b0;
    p.tiles[r] = t1;
    t1 += tiles[i];
    b0 += touched[i];
  }
  for (int r = p.n + tid; r < used; r += TH) {
    p.rows[r] = Kv8Row{-1, 0, 0, 0};
    p.blocks[r + 1] = INT32_MAX;  // behind every item
  }
  for (int t = p.T + tid; t < used_t; t += TH) p.tok_row[t] = -2;
  if (tid == 0) {
    p.blocks[p.n] = total;
    *p.free_count = avail - taken;
    p.used[0] = p.n;
    p.used[1] = p.T;
  }
  if (flags) atomicOr(p.status, flags);
  if (p.T <= kMapHere)
    for (int t = tid; t < p.T; t += TH) map_token(p, scu, t);
}

__global__ __launch_bounds__(256) void kv8_map_kernel(Kv8Plan p) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < p.T) map_token(p, p.cu, t);
}

}  // namespace

hipError_t launch_kv8_step(const Kv8StepArgs& a) {
  const Kv8Plan& p = a.p;
  auto plan = [&](auto kern, int th) {
    hipLaunchKernelGGL(kern, dim3(1), dim3(th), 0, a.stream, p, a.slots, a.lens, a.ntok, a.lens_out);
  };
  if (p.n <= 256 && p.T <= 1024)
    plan(kv8_plan_kernel<256, 1>, 256);
  else if (p.n <= 1024)
    plan(kv8_plan_kernel<1024, 1>, 1024);
  else
    plan(kv8_plan_kernel<1024, kKv8Rows / 1024>, 1024);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.T <= kMapHere) return e;
  hipLaunchKernelGGL(kv8_map_kernel, dim3((p.T + 255) / 256), dim3(256), 0, a.stream, p);
  return hipGetLastError();
}

// --------------------------------------------------------------------- append --

namespace {

// The largest of the 16-bit halves' low 15 bits, both by v_pk_max_u16.
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

// Top bits of the NaN bytes of a word of e4m3.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// Four bytes times 2^k (a factor), rounded anew.
__device__ __forceinline__ uint32_t again4(uint32_t w, float f) {
  return e4m3_pair(__builtin_amdgcn_cvt_f32_fp8(w, 0) * f, __builtin_amdgcn_cvt_f32_fp8(w, 1) * f) |
         e4m3_pair(__builtin_amdgcn_cvt_f32_fp8(w, 2) * f, __builtin_amdgcn_cvt_f32_fp8(w, 3) * f) << 16;
}

}  // namespace

// grid (pages that the step can touch, Hkv, 2), block 256: one page's K (z = 0) or V tile of
// a head. The new rows and the tile's old bytes come into registers; their largest
// magnitudes (as integers: bf16 and e4m3 patterns are in the order of their values) give the
// exponent. A page that is new or whose exponent changes is put together in LDS and written
// whole; otherwise only the new rows' bytes are. An item is 4 keys x 8 dims: 8 bytes of each
// key in K's order, a word of 4 keys for each dim in V's. Bound by latency: the tables, the exponent,
// the old bytes and a barrier one after the other. 64 single tokens of 2 heads of 256 dims 8 us,
// 9.3 where every page is rewritten; 2,899 tokens of 8 heads of 128 dims 10 to 12 us (18 MB). Element
// by element, every page written whole, the 64 tokens took 27 us with a gather of them, where this
// takes 12.
template <int D>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a) {
  constexpr int kChunks = D / 8, kItems = 16 * kChunks, kPer = (kItems + 255) / 256;
  constexpr int kOld = kPage * D / 16 / 256;  // 16-byte pieces of a tile a thread
  __shared__ u32x4 tile4[kPage * D / 16];
  __shared__ uint32_t red[2][4];
  uint8_t* const tile = reinterpret_cast<uint8_t*>(tile4);
  const Kv8Plan& p = a.p;
  const int tid = threadIdx.x, j = blockIdx.y, isv = blockIdx.z;
  const int e = blockIdx.x;
  if (e >= p.blocks[p.n]) return;
  const int r = row_of(p.blocks, p.n, e);
  const Kv8Row row = p.rows[r];
  const int slot = row.slot, len = row.pos, fresh = kv8_tokens(p, row);
  if (fresh == 0) return;
  const int blk = len / kPage + e - p.blocks[r];
  const int first = blk * kPage;
  const int old = max(len - first, 0);                  // tokens that are there
  const int last = min(len + fresh - first, kPage);     // and with the new ones
  const int page = p.table[(size_t)slot * p.max_pages + blk];
  const size_t head = ((size_t)page * 2 + isv) * p.Hkv + j;
  u32x4* const dst = reinterpret_cast<u32x4*>(a.pages + head * (kPage * D));
  const uint16_t* const src = isv ? a.v : a.k;
  const int64_t stride = isv ? a.vs : a.ks;
  // row of token `first` in the packed tensors
  const int64_t row0 = (int64_t)row.cu + first - len;
  const int was = old ? a.exps[head] : 0;

  u32x4 x[kPer][4], ob[kOld];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int it = tid + 256 * i, c = it % kChunks, g = it / kChunks;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int kk = 4 * g + k;
      x[i][k] = (u32x4){0u, 0u, 0u, 0u};
      if (it < kItems && kk >= old && kk < last)
        x[i][k] = *reinterpret_cast<const u32x4*>(src + (row0 + kk) * stride + j * D + 8 * c);
    }
  }
  // bf16 magnitudes of the new rows, e4m3 ones of the old; infinities and NaN do not count
  uint32_t mx2 = 0, mo2 = 0;
  bool nan = false;
  if (old) {
#pragma unroll
    for (int i = 0; i < kOld; ++i) ob[i] = dst[tid + 256 * i];
#pragma unroll
    for (int i = 0; i < kOld; ++i) {
      // the piece's keys: K one (16 dims of it), V four words of four
      const int at = tid + 256 * i;
      const int kkey = at / D * 16 + at % 16;
      const int v0 = at / (2 * D) * 32 + 4 * (at / 16 % 2);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = isv ? old - (v0 + 8 * (w >> 1) + 16 * (w & 1)) : kkey < old ? 4 : 0;
        const uint32_t b = n >= 4 ? ob[i][w] : n <= 0 ? 0u : ob[i][w] & ((1u << (8 * n)) - 1u);
        ob[i][w] = b;  // nothing behind the old rows
        const uint32_t top = nan_bytes(b);
        nan |= top != 0;
        const uint32_t m = b & 0x7f7f7f7fu & ~((top >> 7) * 0xffu);
        mo2 = pk_max(mo2, pk_max(m & 0x00ff00ffu, (m >> 8) & 0x00ff00ffu));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t m = x[i][k][w] & 0x7fff7fffu;
        if ((m & 0x7f80u) == 0x7f80u) {
          nan = true;
          m &= 0xffff0000u;
        }
        if ((m & 0x7f800000u) == 0x7f800000u) {
          nan = true;
          m &= 0xffffu;
        }
        mx2 = pk_max(mx2, m);
      }
  uint32_t both = max(mx2 & 0xffffu, mx2 >> 16) << 8 | max(mo2 & 0xffffu, mo2 >> 16);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t u = __shfl_xor(both, off, 64);
    both = max(both & ~0xffu, u & ~0xffu) | max(both & 0xffu, u & 0xffu);
  }
  const bool wave_nan = __any(nan);
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = both;
    red[1][tid >> 6] = wave_nan;
  }
  __syncthreads();
  uint32_t mx = 0, mo = 0, any_nan = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mx = max(mx, red[0][i] >> 8);
    mo = max(mo, red[0][i] & 0xffu);
    any_nan |= red[1][i];
  }
  const int eo = (int)(int8_t)was;
  const float vold = old ? e4m3_value(mo) * pow2(eo) : 0.f;
  const int en = exponent_of(__float_as_uint(fmaxf(__uint_as_float(mx << 16), vold)));
  const float inv = pow2(-en);
  const bool whole = old == 0 || en != eo;
  if (whole && old) {  // the old rows first, the new ones' bytes over them
    const float f = pow2(eo - en);
#pragma unroll
    for (int i = 0; i < kOld; ++i)
      tile4[tid + 256 * i] =
          (u32x4){again4(ob[i][0], f), again4(ob[i][1], f), again4(ob[i][2], f), again4(ob[i][3], f)};
    __syncthreads();
  }
  uint8_t* const to = whole ? tile : reinterpret_cast<uint8_t*>(dst);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int it = tid + 256 * i, c = it % kChunks, g = it / kChunks;
    if (it >= kItems) break;
    if (old && (4 * g + 3 < old || 4 * g >= last)) continue;
    uint32_t b[4][2];  // per key 8 bytes
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int w = 0; w < 2; ++w)
        b[k][w] = e4m3_pair(bf_lo(x[i][k][2 * w]) * inv, bf_hi(x[i][k][2 * w]) * inv) |
                  e4m3_pair(bf_lo(x[i][k][2 * w + 1]) * inv, bf_hi(x[i][k][2 * w + 1]) * inv) << 16;
    const bool all = old == 0 || (4 * g >= old && 4 * g + 3 < last);  // the item's four keys
    if (isv) {
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const int w = d >> 2, s = 8 * (d & 3);
        uint8_t* const at = to + v_byte(4 * g, 8 * c + d, D);
        if (all) {
          *reinterpret_cast<uint32_t*>(at) =
              ((b[0][w] >> s) & 0xffu) | ((b[1][w] >> s) & 0xffu) << 8 |
              ((b[2][w] >> s) & 0xffu) << 16 | ((b[3][w] >> s) & 0xffu) << 24;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (4 * g + k >= old && 4 * g + k < last) at[k] = (uint8_t)(b[k][w] >> s);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (all || (4 * g + k >= old && 4 * g + k < last))
          *reinterpret_cast<u32x2*>(to + k_byte(4 * g + k, 8 * c, D)) = (u32x2){b[k][0], b[k][1]};
    }
  }
  if (whole) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOld; ++i) dst[tid + 256 * i] = tile4[tid + 256 * i];
  }
  if (tid == 0) a.exps[head] = (en & 0xff) | (any_nan ? kNanFlag : 0);
}

hipError_t launch_kv8_append(const Kv8AppendArgs& a) {
  const Kv8Plan& p = a.p;
  // a row of m tokens touches at most m pages, and at most m / 64 + 2
  const int most = min(p.T, p.T / kPage + 2 * min(p.n, p.T));
  const dim3 grid(most, p.Hkv, 2);
  if (p.D == 256)
    hipLaunchKernelGGL(kv8_append_kernel<256>, grid, dim3(256), 0, a.stream, a);
  else if (p.D == 128)
    hipLaunchKernelGGL(kv8_append_kernel<128>, grid, dim3(256), 0, a.stream, a);
  else
    hipLaunchKernelGGL(kv8_append_kernel<64>, grid, dim3(256), 0, a.stream, a);
  return hipGetLastError();
}

// --------------------------------------------------------------------- gather --

namespace {

// grid (ceil(m / 64) from `from` on, Hkv * D / 32, 2), block 256: 64 places, 32 dims of a head, K
// (z = 0) or V; 8 dims of a place a thread. Places that run through a page, as a sequence's do,
// share the cache lines of V's bytes. 2,899 places of 8 heads of
// 128 dims 8 us (18 MB), 64 of 2 heads 4: latency, the map before the bytes.
__global__ __launch_bounds__(256) void kv8_gather_kernel(Kv8GatherArgs a, int64_t from) {
  const Kv8Plan& p = a.p;
  const int z = blockIdx.z, parts = p.D / 32, j = blockIdx.y / parts;
  const int d = (blockIdx.y - j * parts) * 32 + 8 * (threadIdx.x & 3);
  uint16_t* const out = z ? a.v_out : a.k_out;
  const int64_t t = (from + blockIdx.x) * 64 + (threadIdx.x >> 2);
  if (!out || t >= a.m) return;
  const int place = a.map[t];
  u32x4 o = {0u, 0u, 0u, 0u};
  if (place >= 0 && place < p.num_pages * kPage) {
    const int kk = place & (kPage - 1);
    const size_t head = ((size_t)(place / kPage) * 2 + z) * p.Hkv + j;
    const uint8_t* const tile = a.pages + head * ((size_t)kPage * p.D);
    const float s = pow2((int)(int8_t)a.exps[head]);
    float f[8];
    if (z) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = e4m3_value(tile[v_byte(kk, d + i, p.D)]) * s;
    } else {
      const u32x2 b = *reinterpret_cast<const u32x2*>(tile + k_byte(kk, d, p.D));
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = e4m3_value((b[i >> 2] >> (8 * (i & 3))) & 0xffu) * s;
    }
    // four significant bits: exact in bf16
    o = (u32x4){f2bf2(f[0], f[1]), f2bf2(f[2], f[3]), f2bf2(f[4], f[5]), f2bf2(f[6], f[7])};
  }
  *reinterpret_cast<u32x4*>(out + t * (z ? a.vs : a.ks) + j * p.D + d) = o;
}

}  // namespace

hipError_t launch_kv8_gather(const Kv8GatherArgs& a) {
  const int64_t groups = ((int64_t)a.m + 63) / 64;
  constexpr int64_t kGroups = 1 << 16;
  for (int64_t g = 0; g < groups; g += kGroups) {
    const dim3 grid((unsigned)(groups - g < kGroups ? groups - g : kGroups), a.p.Hkv * (a.p.D / 32), 2);
    hipLaunchKernelGGL(kv8_gather_kernel, grid, dim3(256), 0, a.stream, a, g);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace gdn
