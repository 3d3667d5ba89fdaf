// KV pages in 8 bits on sm_100a: append (rotation and quantisation on the way), read-back, and attention over the pages.
// The page and why it is laid out so: st_kv8.cuh.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "../../include/statetree_b200.h"
#include "st_host.h"
#include "st_kv8.cuh"

namespace {
using namespace st;

// ------------------------------------------------------------------------------------------------ append
// Keys (normalised and rotated on the way, in fp32, one rounding to e4m3 at the end), values, and the queries of the same tokens
// (normalised and rotated into q_out).  A warp (or two) owns one unit (page, head, K or V) for the launch and takes every token of the
// call that goes to the page, so the result does not depend on any order:
//     e' = the smallest exponent that holds the new rows; the page's old one if that is larger and the page does not start anew
//     new rows are rounded at e', the others again at e' if it differs from the old exponent, or cleared if row 0 is among the new
// Which warp: the last token of the call in a page leads it.
//   SCAN  (calls of up to SCAN_MAX tokens, about where the two meet: keys and values of 16, 256, 512 sequences with a token each 4.6,
//         9.2, 17.5 us so, 8.3, 10.5, 16.4 with marks; 512 tokens of one 10.9 and 11.6) a warp per (token, unit) walks the call's slots
//         and finds out itself
//   else  kv8_mark_kernel leaves every row's and page's last token in `marks`; a CTA takes up to sixteen tokens of the call, clears the
//         marks of the pages they lead and writes all units of those (fewer tokens in shorter calls, which may lead a page each: 1024
//         sequences 92 us with sixteen, 25 with one).  At D = 128 two warps share a unit: with half the values a lane, 24 warps find
//         room on an SM for 16 (32764 tokens 163 us for 179, with 2 KV and 16 query heads 87 for 116; four warps a unit 171: before
//         the keys' rotation became a closer one)
// One token (8 KV heads, 32 query heads) 4.2 us, bound by look-ups that follow one another; 32764 tokens 167 us (755 MB), of which keys
// and values take 81 (a chain of look-ups and 40 % of the issue slots) and the queries 86 (HBM).
// Same slot twice: the last one counts in both.  Values that are not finite are stored as the largest of their sign (infinities) or
// as zero (NaN), and flagged in *bad.
constexpr int SCAN_MAX = 384;

struct Append8 {
  const uint16_t* K; const uint16_t* V; const uint16_t* Q;
  long long ks, vs, qs, qos;
  const long long* slot;
  uint8_t* kv; int8_t* exps;
  long long nblocks;
  const long long* pos; long long pos_step; long long max_pos;
  const float* cos_t; const float* sin_t;
  const uint16_t* wq; const uint16_t* wk;
  uint16_t* q_out;
  int* marks; int* bad;
  int N, H, Hq;
  int run;                                         // tokens of the call that a CTA looks at (without SCAN), up to sixteen
  int q_cta, q_units, q_steps;                     // first CTA that works on queries; warps per token, groups of heads per warp
  float eps;
  int pairs;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[16], int at) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[at + 2 * i] = __uint_as_float(w[i] << 16);
    f[at + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// A lane's sixteen values of a row: dims 8c .. 8c + 7 (f[0..7]) and D/2 + 8c .. (f[8..15]), c = lane % (D / 16): both partners of
// either rotation lie in one lane.
template <int D>
__device__ __forceinline__ float row_rms(const float (&f)[16], float eps) {
  constexpr int LPR = D / 16;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
  return __frsqrt_rn(ss * (1.f / D) + eps);
}
// the row times the norm weights: exact, both are BF16
__device__ __forceinline__ void row_weights(float (&f)[16], const uint4 (&w)[2]) {
  float g[16];
  unpack8(w[0], g, 0);
  unpack8(w[1], g, 8);
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] *= g[i];
}
template <int D>
__device__ __forceinline__ void norm_weights(uint4 (&w)[2], const uint16_t* at, int c) {
  w[0] = *reinterpret_cast<const uint4*>(at + 8 * c);
  w[1] = *reinterpret_cast<const uint4*>(at + D / 2 + 8 * c);
}
struct Turn { float cs[8], sn[8]; };               // of the lane's eight pairs
template <int D>
__device__ __forceinline__ void load_turn(Turn& t, const float* ct, const float* st, int pairs, int c) {
  const int p0 = pairs ? 4 * c : 8 * c, p1 = pairs ? D / 4 + 4 * c : 8 * c + 4;
  *reinterpret_cast<float4*>(t.cs) = *reinterpret_cast<const float4*>(ct + p0);
  *reinterpret_cast<float4*>(t.cs + 4) = *reinterpret_cast<const float4*>(ct + p1);
  *reinterpret_cast<float4*>(t.sn) = *reinterpret_cast<const float4*>(st + p0);
  *reinterpret_cast<float4*>(t.sn + 4) = *reinterpret_cast<const float4*>(st + p1);
}
// a * b - c * d, with the rounding of c * d taken out of the difference: 1.5 steps of the result at most, however much cancels
__device__ __forceinline__ float diff_of_products(float a, float b, float c, float d) {
  const float p = c * d;
  return fmaf(a, b, -p) + fmaf(-c, d, p);
}
// CLOSE: for keys, so that their codes are the exact value's more often (3 x 8.4 million normalised and rotated keys: 22 codes are not, with
// two plain roundings each 33; 32764 tokens 167 us for 163)
template <bool CLOSE>
__device__ __forceinline__ void rotate_pair(float& a, float& b, float cs, float sn) {
  const float x = a, y = b;
  a = CLOSE ? diff_of_products(x, cs, y, sn) : x * cs - y * sn;
  b = CLOSE ? diff_of_products(x, sn, -y, cs) : x * sn + y * cs;
}
template <bool CLOSE>
__device__ __forceinline__ void row_rotate(float (&f)[16], const Turn& t, int pairs) {
  if (pairs) {
#pragma unroll
    for (int i = 0; i < 8; ++i) rotate_pair<CLOSE>(f[2 * i], f[2 * i + 1], t.cs[i], t.sn[i]);      // pair i of the lane
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) rotate_pair<CLOSE>(f[i], f[8 + i], t.cs[i], t.sn[i]);
  }
}
__device__ __forceinline__ long long table_row(const Append8& a, long long token) {
  const long long p = a.pos[token * a.pos_step];
  return p < 0 ? 0 : (p >= a.max_pos ? a.max_pos - 1 : p);
}

// the smallest e in [E8_MIN, E8_MAX] with top <= 448 * 2^e (448 = 1.75 * 2^8), top >= 0 and finite
__device__ __forceinline__ int exp_for(float top) {
  const uint32_t b = __float_as_uint(top);
  return page8_exp((int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {        // round to nearest even, |x| <= 448
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 e4m3_eight(const float* f, float down) {
  uint2 u;
  u.x = e4m3_pair(f[0] * down, f[1] * down) | e4m3_pair(f[2] * down, f[3] * down) << 16;
  u.y = e4m3_pair(f[4] * down, f[5] * down) | e4m3_pair(f[6] * down, f[7] * down) << 16;
  return u;
}
__device__ __forceinline__ uint2 rescale_eight(uint2 u, float up, float down) {
  float f[8];
  uint32_t p[4];
  codes_to_bf16(u.x, p[0], p[1]);
  codes_to_bf16(u.y, p[2], p[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = codes_value(p[i], up);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
  return e4m3_eight(f, down);
}

// the largest of a value of each of the WPU warps that share a unit; `at` is theirs (nobody writes it again before all have read it)
template <int WPU>
__device__ __forceinline__ uint32_t over_warps_max(uint32_t v, uint32_t* at, int warp, int lane) {
  if (WPU == 1) return v;
  if (lane == 0) at[warp % WPU] = v;
  asm volatile("bar.sync %0, %1;" :: "r"(1 + warp / WPU), "n"(32 * WPU) : "memory");
#pragma unroll
  for (int k = 0; k < WPU; ++k) v = max(v, at[k]);
  return v;
}
// one unit: lane r < 16 holds in `tok` the token that goes to row r, -1 = none; at least one row has a token.  WPU warps share it, some
// rows each; `share`: 2 * WPU words of theirs, others than for the unit before
template <int D, int WPU>
__device__ __forceinline__ void append_unit(const Append8& a, long long page, int h, int kvi, int tok, int warp, int lane, uint32_t* share) {
  constexpr int LPR = D / 16, RPI = 32 / LPR, ITER = PAGE / RPI / WPU;
  const int row0 = warp % WPU * (ITER * RPI);
  const unsigned rows = __ballot_sync(FULL, lane < PAGE && tok >= 0);
  const int c = lane % LPR;
  const uint16_t* const src = (kvi ? a.V : a.K) + (size_t)h * D + 8 * c;
  const long long step = kvi ? a.vs : a.ks;
  uint4 raw[ITER][2];
  int mine[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    mine[i] = __shfl_sync(FULL, tok, row0 + i * RPI + lane / LPR);
    raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
    if (mine[i] >= 0) {
      const uint16_t* p = src + (long long)mine[i] * step;
      raw[i][0] = *reinterpret_cast<const uint4*>(p);
      raw[i][1] = *reinterpret_cast<const uint4*>(p + D / 2);
    }
  }
  int8_t* const exp_at = a.exps + ((size_t)page * a.H + h) * 2 + kvi;
  const bool anew = rows & 1u;
  const int was = anew ? E8_MIN : page8_exp(*exp_at);
  float f[ITER][16];
  uint4 w[2];
  if (kvi == 0 && a.wk) norm_weights<D>(w, a.wk, c);
  uint32_t most = 0;                               // bits of the largest magnitude: NaN above infinity above the finite ones
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    unpack8(raw[i][0], f[i], 0);
    unpack8(raw[i][1], f[i], 8);
    if (kvi == 0) {                                // (the row's factor last: a rotation does not change it, and it rounds once)
      const float r = a.wk ? row_rms<D>(f[i], a.eps) : 1.f;
      if (a.wk) row_weights(f[i], w);
      if (a.cos_t && mine[i] >= 0) {
        const long long at = table_row(a, mine[i]) * (D / 2);
        Turn t;
        load_turn<D>(t, a.cos_t + at, a.sin_t + at, a.pairs, c);
        row_rotate<true>(f[i], t, a.pairs);
      }
      if (a.wk)
#pragma unroll
        for (int k = 0; k < 16; ++k) f[i][k] *= r;
    }
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) m = max(m, __float_as_uint(f[i][k]) & 0x7FFFFFFFu);
    if (mine[i] >= 0) most = max(most, m);         // (norm and rotation can make NaN of a row without a token: 0 * rsqrt(0))
  }
  most = over_warps_max<WPU>(__reduce_max_sync(FULL, most), share, warp, lane);
  const bool odd = most > __float_as_uint(448.f * pow2i(E8_MAX));        // (a value that is not finite, or beyond the format)
  float top = __uint_as_float(most);
  if (odd) {
    top = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float m = fabsf(f[i][k]);
        top = fmaxf(top, m < INFINITY ? m : 0.f);
        if (m != m) f[i][k] = 0.f;
      }
    top = __uint_as_float(over_warps_max<WPU>(__reduce_max_sync(FULL, __float_as_uint(top)), share + WPU, warp, lane));
  }
  const int e = max(was, exp_for(top));
  const float down = pow2i(-e), up = pow2i(20 + was);
  uint8_t* const unit = a.kv + page8_off<D>(page, a.H, h, kvi);
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int r = row0 + i * RPI + lane / LPR;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int d = half * (D / 2) + 8 * c;
      uint2* const at = reinterpret_cast<uint2*>(unit + r * D + 16 * piece8<D>(r, d >> 4) + (d & 8));
      if (mine[i] >= 0) *at = e4m3_eight(f[i] + 8 * half, down);
      else if (anew) *at = make_uint2(0, 0);
      else if (e != was) *at = rescale_eight(*at, up, down);
    }
  }
  __syncwarp();                                    // (every lane has read the old exponent, the other warps' before they met)
  if (lane == 0 && row0 == 0 && (anew || e != was)) *exp_at = (int8_t)e;
  if (odd && lane == 0) *a.bad = 1;
}

// A warp takes q_steps groups of 32 / (D / 16) heads of one token: its row of the tables and the norm weights are read once
template <int D, int AHEAD>
__device__ __forceinline__ void rotate_queries(const Append8& a, long long unit, int lane) {
  constexpr int LPR = D / 16, RPI = 32 / LPR;
  const long long token = unit / a.q_units;
  if (token >= a.N) return;
  const int c = lane % LPR, h0 = (int)(unit % a.q_units) * a.q_steps * RPI, h1 = min(a.Hq, h0 + a.q_steps * RPI);
  const uint16_t* const src = a.Q + token * a.qs + 8 * c;
  uint16_t* const dst = a.q_out + token * a.qos + 8 * c;
  uint4 w[2];
  Turn t;
  if (a.cos_t) {
    const long long at = table_row(a, token) * (D / 2);
    load_turn<D>(t, a.cos_t + at, a.sin_t + at, a.pairs, c);
  }
  if (a.wq) norm_weights<D>(w, a.wq, c);
  for (int h = h0; h < h1; h += AHEAD * RPI) {
    uint4 raw[AHEAD][2];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int mine = h + i * RPI + lane / LPR;
      if (mine < h1) {
        raw[i][0] = *reinterpret_cast<const uint4*>(src + (size_t)mine * D);
        raw[i][1] = *reinterpret_cast<const uint4*>(src + (size_t)mine * D + D / 2);
      }
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (h + i * RPI >= h1) break;
      const int mine = h + i * RPI + lane / LPR;
      float f[16];
      unpack8(raw[i][0], f, 0);
      unpack8(raw[i][1], f, 8);
      const float r = a.wq ? row_rms<D>(f, a.eps) : 1.f;
      if (a.wq) row_weights(f, w);
      if (a.cos_t) row_rotate<false>(f, t, a.pairs);
#pragma unroll
      for (int k = 0; k < 16; ++k) f[k] *= r;
      if (mine < h1) {
        uint4* const o = reinterpret_cast<uint4*>(dst + (size_t)mine * D);
        o[0] = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
        *reinterpret_cast<uint4*>(dst + (size_t)mine * D + D / 2) =
            make_uint4(pack_bf16(f[8], f[9]), pack_bf16(f[10], f[11]), pack_bf16(f[12], f[13]), pack_bf16(f[14], f[15]));
      }
    }
  }
}

__device__ __forceinline__ bool slot_ok(const Append8& a, long long s) { return s >= 0 && s / PAGE < a.nblocks; }

__global__ void __launch_bounds__(256) kv8_mark_kernel(const Append8 a) {
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.N) return;
  const long long s = a.slot[i];
  if (!slot_ok(a, s)) return;
  atomicMax(a.marks + s, i + 1);
  atomicMax(a.marks + a.nblocks * PAGE + s / PAGE, i + 1);
}

template <int D, bool SCAN>
__global__ void __launch_bounds__(256, SCAN ? 2 : 3) kv8_append_kernel(const Append8 a) {
  constexpr int WPU = SCAN ? 1 : D / 64;
  __shared__ int s_row[PAGE][PAGE];
  __shared__ long long s_page[PAGE];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, units = 2 * a.H;
  if ((int)blockIdx.x >= a.q_cta) {
    rotate_queries<D, SCAN ? 4 : 2>(a, (long long)((int)blockIdx.x - a.q_cta) * 8 + warp, lane);
    return;
  }
  if (SCAN) {
    const long long w = (long long)blockIdx.x * 8 + warp;
    const int i = (int)(w / units), u = (int)(w % units);
    if (i >= a.N) return;
    const long long s = a.slot[i];
    if (!slot_ok(a, s)) return;
    const long long page = s / PAGE;
    int* const row = s_row[warp];
    if (lane < PAGE) row[lane] = -1;
    __syncwarp();
    bool later = false;
    for (int j = lane; j < a.N; j += 32) {
      const long long t = a.slot[j];
      if (t >= 0 && t / PAGE == page) {
        later |= j > i;
        atomicMax(row + (int)(t % PAGE), j);
      }
    }
    if (__any_sync(FULL, later)) return;           // (a later token leads the page)
    __syncwarp();
    append_unit<D, WPU>(a, page, u >> 1, u & 1, lane < PAGE ? row[lane] : -1, warp, lane, nullptr);
  } else {
    if (warp == 0) {
      const int i = (int)blockIdx.x * a.run + lane;
      const long long s = lane < a.run && i < a.N ? a.slot[i] : -1;
      const bool leads = slot_ok(a, s) && a.marks[a.nblocks * PAGE + s / PAGE] == i + 1;
      if (lane < PAGE) s_page[lane] = -1;
      __syncwarp();
      int n = 0;
      for (unsigned left = __ballot_sync(FULL, leads); left; left &= left - 1, ++n) {
        const long long page = __shfl_sync(FULL, s, __ffs(left) - 1) / PAGE;
        if (lane < PAGE) {                         // (nobody else reads these marks: the page's other tokens do not lead it)
          s_row[n][lane] = a.marks[page * PAGE + lane] - 1;
          a.marks[page * PAGE + lane] = 0;
        }
        if (lane == 0) {
          s_page[n] = page;
          a.marks[a.nblocks * PAGE + page] = 0;
        }
      }
    }
    __syncthreads();
    // (keys of all heads, then values: every warp has some of both)
    __shared__ uint32_t s_share[8 / WPU][2][2 * WPU];
    int turn = 0;
    for (int n = 0; n < PAGE && s_page[n] >= 0; ++n) {
      const int tok = lane < PAGE ? s_row[n][lane] : -1;
      for (int u = warp / WPU; u < units; u += 8 / WPU, turn ^= 1)
        append_unit<D, WPU>(a, s_page[n], u < a.H ? u : u - a.H, u >= a.H, tok, warp, lane, s_share[warp / WPU][turn]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ read-back
// listed pages (blocks != nullptr) or every page -> dense BF16 [n, 16, H, D]; sixteen values per thread
template <int D>
__global__ void __launch_bounds__(256) kv8_dequant_kernel(const uint8_t* __restrict__ kv, const int8_t* __restrict__ exps,
                                                          long long nblocks, int H, const int* __restrict__ blocks, long long n,
                                                          uint16_t* __restrict__ Kd, uint16_t* __restrict__ Vd) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int PIECES = PAGE * D / 16;            // of a unit
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long unit = x / PIECES;
  if (unit >= n * H * 2) return;
  const int p = (int)(x % PIECES), r = p / (D / 16), c = p % (D / 16), kvi = (int)(unit & 1), h = (int)((unit >> 1) % H);
  const long long i = (unit >> 1) / H, blk = blocks ? (long long)blocks[i] : i;
  uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (blk >= 0 && blk < nblocks) {
    const uint4 u = *reinterpret_cast<const uint4*>(kv + page8_off<D>(blk, H, h, kvi) + r * D + 16 * piece8<D>(r, c));
    const float up = pow2i(20 + page8_exp(exps[((size_t)blk * H + h) * 2 + kvi]));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t b[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t p01, p23;
      codes_to_bf16(w[k], p01, p23);
      const float2 lo = codes_value(p01, up), hi = codes_value(p23, up);
      b[2 * k] = pack_bf16(lo.x, lo.y);
      b[2 * k + 1] = pack_bf16(hi.x, hi.y);
    }
    o[0] = make_uint4(b[0], b[1], b[2], b[3]);
    o[1] = make_uint4(b[4], b[5], b[6], b[7]);
  }
  uint4* const out = reinterpret_cast<uint4*>((kvi ? Vd : Kd) + (((size_t)i * PAGE + r) * H + h) * D + 16 * c);
  out[0] = o[0];
  out[1] = o[1];
}

// ------------------------------------------------------------------------------------------------ attention, one token per sequence
// Orientation.  A decode step has few query heads per KV head, so the heads of a group go on the 8-wide N side of mma.m16n8k16 and
// tokens / dims on the 16-wide M side (groups of more than eight take a CTA per eight heads):
//     S^T [16 tokens x 8 heads] = K [16 tokens x D dims] . Q^T        O^T [D dims x 8 heads] += V^T [D dims x 16 tokens] . P^T
// The order of the k index is free as long as both operands agree on it: lane (g, t) = (lane / 4, lane % 4) takes for keys the
// 16-byte pieces t and t + 4 of rows g and g + 8 as they lie in the page, four dims per MMA, and q in the same order; for values the
// piece g of tokens 2t, 2t + 1, 2t + 8, 2t + 9, two dims per MMA, the codes of two tokens being paired by a byte permute.  So codes go
// to fragments without a transposition through memory.
//
// Types and scales.  An e4m3 code is an FP16 number exactly, and one instruction converts two (as BF16 patterns they took 1.75
// integer operations each, and the integer pipe, 64 lanes a cycle and SM, was the limit: 64 sequences of up to 8192 tokens 118 us).
// q is scaled by a power of two per head so that FP16 holds its eight bits (of values down to 2^-28 of the head's largest).  The
// exponent of a page's keys joins the softmax scale.  That of its values joins the exponent of its probabilities: with x = score +
// exponent (base 2) and a running reference r, P = 2^(x - r) <= 2^15 is rounded to FP16 (2^-11 of each at most, and 2^-32 of the
// largest), and the sum of the probabilities takes the exponent out again, per page, in fp32.
//
// A head's reference r stays between 7 and 15 below its largest x so far: it is raised when a page holds an x more than 15 above it,
// one vote per page, a rescale only then.
//
// Work split: grid = sequences x KV heads x head blocks x splits; a CTA's pages go round-robin to its warps, each of which streams its
// own through a private ring of bulk copies (a page of one head is contiguous, 2 * 16 * D bytes), so there is no barrier in the loop.
// Block-table entries and exponents come 32 pages at a time, one batch ahead.  The splits of a unit join through distributed shared memory,
// as a cluster, or through memory in a second kernel (joins8).
// Measured (32 query heads, 8 KV heads, D = 128, in a graph): 64 sequences of up to 8192 tokens 90 us = 5.9 TB/s, one of 61003 23.0 us, one
// of 1000 5.0-5.4 us.
__device__ __forceinline__ float over_rows_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(FULL, v, 4));
  v = fmaxf(v, __shfl_xor_sync(FULL, v, 8));
  return fmaxf(v, __shfl_xor_sync(FULL, v, 16));
}
__device__ __forceinline__ float over_rows_sum(float v) {
  v += __shfl_xor_sync(FULL, v, 4);
  v += __shfl_xor_sync(FULL, v, 8);
  return v + __shfl_xor_sync(FULL, v, 16);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// CHUNK: several queries per sequence.  The eight columns are then rows (query, head) of the sequence's n * G, each with keys of its own
// [lo, hi], and a tile of eight of them is looked up as in the chunk kernel; else they are heads of the one query.
constexpr int JOIN8 = 8;                                          // splits that one cluster joins at most
template <int D, int NW, int STG, bool CHUNK>
__global__ void __launch_bounds__(NW * 32, 16 / NW) kv8_attn_kernel(const Attn8 a, const Parts8 parts, int* status) {
  constexpr int PB = 2 * PAGE * D, KT = D / 16, VT = D / 16;             // bytes of a page, MMAs of its keys and of its values
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + NW * STG * PB);
  float2* const facs = reinterpret_cast<float2*>(bars + NW * STG);       // (softmax scale with the keys' exponent, values' exponent)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int G = a.Hq / a.H, blocks_of_heads = (G + 7) / 8;
  const int split = blockIdx.x % parts.splits;
  int rest = blockIdx.x / parts.splits;
  int kvh, seq, heads, first_head, first_row = 0;                 // heads: columns in use
  Rows8 w;
  if (CHUNK) {
    pdl_wait();
    pdl_launch_dependents();
    kvh = rest % a.H;
    if (!find_rows<8>(a, G, rest / a.H, lane, w)) return;
    seq = w.b;
    heads = w.rows;
    first_head = kvh * G;
    first_row = w.row0;
  } else {
    const int hb = rest % blocks_of_heads;
    rest /= blocks_of_heads;
    kvh = rest % a.H;
    seq = rest / a.H;
    heads = min(8, G - 8 * hb);
    first_head = kvh * G + 8 * hb;
  }
  // column c: query (of q) and head
  auto token_of = [&](int c) { return CHUNK ? w.first + (first_row + c) / G : seq; };
  auto head_of = [&](int c) { return CHUNK ? first_head + (first_row + c) % G : first_head + c; };
  uint8_t* const ring = smem + warp * STG * PB;
  uint64_t* const bar = bars + warp * STG;
  float2* const fac = facs + warp * STG;
  if (lane == 0) {
    for (int s = 0; s < STG; ++s) mbar_init(bar + s, 1);
    fence_barrier_init();
  }
  const uint64_t stream_policy = CHUNK ? policy_evict_last() : policy_evict_first();      // (other rows of a chunk read the same pages)
  if (!CHUNK) {
    pdl_wait();
    pdl_launch_dependents();
  }

  const int len = CHUNK ? w.len : a.lens[seq], start = CHUNK ? w.start : a.starts ? max(a.starts[seq], 0) : 0;
  // keys [lo, end) of the columns together; column c sees [max(start, p - window + 1), p], p its query's position
  const int p0 = CHUNK ? len - w.n + first_row / G : len - 1, p1 = CHUNK ? len - w.n + (first_row + heads - 1) / G : len - 1;
  const int lo = a.window > 0 ? max(start, p0 - a.window + 1) : start, end = p1 + 1;
  const int lo_all = a.window > 0 ? max(start, p1 - a.window + 1) : start, end_all = p0 + 1;      // keys that all columns see
  uint32_t qf[KT][2];
  {
    const int c = g < heads ? g : 0;
    const uint16_t* const qrow = a.q + (size_t)token_of(c) * a.q_stride + (size_t)head_of(c) * D;
#pragma unroll
    for (int p = 0; p < D / 64; ++p) {
      const uint4* const at = reinterpret_cast<const uint4*>(qrow + 16 * (t + 4 * p));
      const uint4 u = at[0], v = at[1];
      qf[4 * p][0] = u.x; qf[4 * p][1] = u.y; qf[4 * p + 1][0] = u.z; qf[4 * p + 1][1] = u.w;
      qf[4 * p + 2][0] = v.x; qf[4 * p + 2][1] = v.y; qf[4 * p + 3][0] = v.z; qf[4 * p + 3][1] = v.w;
    }
  }
  const int first_page = lo / PAGE;
  const int end_page = end > lo ? min((end - 1) / PAGE + 1, a.table_width) : 0;
  const int per_split = max(parts.min_pages, (end_page - first_page + parts.splits - 1) / parts.splits);
  const int lo_page = first_page + split * per_split, hi_page = min(end_page, lo_page + per_split);
  const int my_first = lo_page + warp;
  const int my_count = hi_page > my_first ? (hi_page - my_first + NW - 1) / NW : 0;

  const int* const my_table = a.table + (size_t)seq * a.table_stride + my_first;
  auto entry = [&](int i) {
    int e = i + lane < my_count ? __ldg(my_table + (long long)(i + lane) * NW) : 0;
    return e < 0 ? 0 : (int)min((long long)e, a.nblocks - 1);
  };
  auto factors = [&](int e) {                                     // (both exponents of the page in one load)
    const uint32_t x = __ldg(reinterpret_cast<const uint16_t*>(a.exps) + (size_t)e * a.H + kvh);
    return make_float2(a.scale_log2 * pow2i(page8_exp((int8_t)(x & 0xFF))), (float)page8_exp((int8_t)(x >> 8)));
  };
  int now = entry(0), next = entry(32);
  float2 now_f = factors(now), next_f = now_f;
  const uint8_t* const head_pages = a.kv + page8_off<D>(0, a.H, kvh, 0);
  const size_t page_step = (size_t)a.H * PB;
  auto fetch = [&](int i, int s) {                                // this warp's i-th page -> stage s (whole warp, i in order)
    if ((i & 31) == 0 && i > 0) {
      now = next;
      now_f = next_f;
      next = entry(i + 32);
    }
    if ((i & 31) == 16) next_f = factors(next);
    const int blk = __shfl_sync(FULL, now, i & 31);
    const float2 f = make_float2(__shfl_sync(FULL, now_f.x, i & 31), __shfl_sync(FULL, now_f.y, i & 31));
    if (elect_one()) {
      fac[s] = f;
      mbar_expect_tx(bar + s, PB);
      bulk_g2s(ring + s * PB, head_pages + blk * page_step, PB, bar + s, stream_policy);
    }
  };
  __syncwarp();
#pragma unroll
  for (int i = 0; i < STG; ++i)
    if (i < my_count) fetch(i, i);
  // ---- q as FP16, head g times 2^(13 - exponent of its largest); columns beyond the heads are zero
  float qs0, qs1;                                                 // what undoes it for this lane's score columns, heads 2t, 2t + 1
  {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) most = max(most, max(qf[k][i] << 16 & 0x7FFF0000u, qf[k][i] & 0x7FFF0000u));
    most = max(most, __shfl_xor_sync(FULL, most, 1));
    most = max(most, __shfl_xor_sync(FULL, most, 2));
    const int e = q_exp(most);
    const float down = pow2i(-e);
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qf[k][i] = g < heads ? pack_f16(__uint_as_float(qf[k][i] << 16) * down, __uint_as_float(qf[k][i] & 0xFFFF0000u) * down) : 0u;
    qs0 = pow2i(__shfl_sync(FULL, e, 8 * t));
    qs1 = pow2i(__shfl_sync(FULL, e, 8 * t + 4));
  }
  const bool head0 = 2 * t < heads, head1 = 2 * t + 1 < heads;
  // (a reference is finite from the start: what is hidden, or below fp32, then is 0 and not -inf - -inf; no head: probabilities are 0)
  float m0 = head0 ? -FLT_MAX : 1e30f, m1 = head1 ? -FLT_MAX : 1e30f, l0 = 0.f, l1 = 0.f;
  float acc[VT][4];                                               // MMA j: [0], [1] dim D/8 g + 2j, [2], [3] the next; heads 2t, 2t + 1
#pragma unroll
  for (int j = 0; j < VT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  bool gave_up = false;
  __syncwarp();

  int s = 0;
  uint32_t phase = 0;
  for (int i = 0, page = my_first; i < my_count; ++i, page += NW) {
    if (!mbar_wait(bar + s, phase)) {
      if (lane == 0) atomicExch(status, ERR_WAIT_FULL);
      for (int k = i + 1; k < min(my_count, i + STG); ++k)        // let the copies still in flight land
        (void)mbar_wait(bar + k % STG, (uint32_t)(k / STG) & 1u);
      gave_up = true;
      break;
    }
    const uint8_t* const pg = ring + s * PB;
    const float2 f = fac[s];
    float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < D / 64; ++p) {
      const uint8_t* const at = pg + g * D + 16 * piece8<D>(g, t + 4 * p);
      const uint4 u = *reinterpret_cast<const uint4*>(at), v = *reinterpret_cast<const uint4*>(at + 8 * D);
      const uint32_t wu[4] = {u.x, u.y, u.z, u.w}, wv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mma_f16(k & 1 ? sd : sc, f16_low(wu[k]), f16_low(wv[k]), f16_high(wu[k]), f16_high(wv[k]), qf[4 * p + k][0], qf[4 * p + k][1]);
    }
    const float c0 = fminf(f.x * qs0, 3e38f), c1 = fminf(f.x * qs1, 3e38f);
    float x00 = fmaf(sc[0] + sd[0], c0, f.y), x01 = fmaf(sc[1] + sd[1], c1, f.y);
    float x10 = fmaf(sc[2] + sd[2], c0, f.y), x11 = fmaf(sc[3] + sd[3], c1, f.y);
    const int t0 = page * PAGE;
    if (t0 < lo_all || t0 + PAGE > end_all) {                     // an edge page: tokens that a column does not see
      const int tok = t0 + g;
      if (CHUNK) {
        const int h0 = len - w.n + (first_row + 2 * t) / G, h1 = len - w.n + (first_row + 2 * t + 1) / G;       // last key of a column
        const int g0 = a.window > 0 ? max(start, h0 - a.window + 1) : start, g1 = a.window > 0 ? max(start, h1 - a.window + 1) : start;
        if (tok < g0 || tok > h0) x00 = -INFINITY;
        if (tok < g1 || tok > h1) x01 = -INFINITY;
        if (tok + 8 < g0 || tok + 8 > h0) x10 = -INFINITY;
        if (tok + 8 < g1 || tok + 8 > h1) x11 = -INFINITY;
      } else {
        if (tok < lo || tok >= end) x00 = x01 = -INFINITY;
        if (tok + 8 < lo || tok + 8 >= end) x10 = x11 = -INFINITY;
      }
    }
    const float top0 = fmaxf(x00, x10), top1 = fmaxf(x01, x11);
    if (__any_sync(FULL, top0 > m0 + RAISE8 || top1 > m1 + RAISE8)) {
      const float n0 = fmaxf(m0, over_rows_max(top0) - UNDER8), n1 = fmaxf(m1, over_rows_max(top1) - UNDER8);
      const float f0 = n0 == m0 ? 1.f : ex2(m0 - n0), f1 = n1 == m1 ? 1.f : ex2(m1 - n1);
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int j = 0; j < VT; ++j) { acc[j][0] *= f0; acc[j][1] *= f1; acc[j][2] *= f0; acc[j][3] *= f1; }
      m0 = n0;
      m1 = n1;
    }
    const float p00 = ex2(x00 - m0), p01 = ex2(x01 - m1), p10 = ex2(x10 - m0), p11 = ex2(x11 - m1), out = ex2(-f.y);
    l0 = fmaf(p00 + p10, out, l0);
    l1 = fmaf(p01 + p11, out, l1);
    const uint32_t b0 = movmatrix_t(pack_f16(p00, p01)), b1 = movmatrix_t(pack_f16(p10, p11));
    const uint8_t* const vp = pg + PAGE * D;
    constexpr int WORDS = D / 32;                                 // of a lane's dims of one token: D / 8 codes
    uint32_t w[4][WORDS];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = 2 * t + (k & 1) + 8 * (k >> 1);
      if (D == 128) {
        const uint4 u = *reinterpret_cast<const uint4*>(vp + r * D + 16 * piece8<D>(r, g));
        w[k][0] = u.x; w[k][1] = u.y; w[k][WORDS > 2 ? 2 : 0] = u.z; w[k][WORDS > 2 ? 3 : 0] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(vp + r * D + 8 * g);
        w[k][0] = u.x; w[k][1] = u.y;
      }
    }
#pragma unroll
    for (int k = 0; k < WORDS; ++k)
#pragma unroll
      for (int d = 0; d < 2; ++d) {                               // dims 4k + 2d, 4k + 2d + 1 of the lane
        const uint32_t u = __byte_perm(w[0][k], w[1][k], d ? 0x7362 : 0x5140), v = __byte_perm(w[2][k], w[3][k], d ? 0x7362 : 0x5140);
        mma_f16(acc[2 * k + d], f16_low(u), f16_high(u), f16_low(v), f16_high(v), b0, b1);
      }
    __syncwarp();                                                 // every lane has read this stage
    if (i + STG < my_count) {
      fence_proxy_async();
      fetch(i + STG, s);
    }
    if (++s == STG) {
      s = 0;
      phase ^= 1u;
    }
  }
  if (gave_up) { m0 = m1 = -FLT_MAX; l0 = l1 = 0.f; }
  l0 = over_rows_sum(l0);
  l1 = over_rows_sum(l1);
  if (m0 == -FLT_MAX && l0 == 0.f) m0 = -INFINITY;                // nothing seen (a sum that is not a number stays one)
  if (m1 == -FLT_MAX && l1 == 0.f) m1 = -INFINITY;

  // ---- the CTA's warps together.  The rings are idle now; each warp parks (O^T, r, l) of its heads there.
  __syncthreads();
  constexpr int ROW = D + 2, PER_WARP = 8 * ROW;
  static_assert((NW + 1) * PER_WARP * 4 <= NW * STG * PB, "parked partials must fit in the rings");
  float* const park = reinterpret_cast<float*>(smem);
  float* const mine = park + warp * PER_WARP;
#pragma unroll
  for (int j = 0; j < VT; ++j) {
    const int d = D / 8 * g + 2 * j;
    if (head0) *reinterpret_cast<float2*>(mine + 2 * t * ROW + d) = make_float2(acc[j][0], acc[j][2]);
    if (head1) *reinterpret_cast<float2*>(mine + (2 * t + 1) * ROW + d) = make_float2(acc[j][1], acc[j][3]);
  }
  if (g == 0) {
    if (head0) *reinterpret_cast<float2*>(mine + 2 * t * ROW + D) = make_float2(m0, l0);
    if (head1) *reinterpret_cast<float2*>(mine + (2 * t + 1) * ROW + D) = make_float2(m1, l1);
  }
  __syncthreads();
  const bool joined = parts.splits > 1 && parts.o == nullptr;     // the splits of a unit are one cluster
  float* const sum = park + NW * PER_WARP;
  for (int e = threadIdx.x; e < heads * D; e += NW * 32) {
    const int h = e / D, d = e % D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, park[w * PER_WARP + h * ROW + D]);
    float den = 0.f, num = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* const pw = park + w * PER_WARP + h * ROW;
      if (pw[D] == -INFINITY) continue;                           // a warp that saw nothing
      const float f = ex2(pw[D] - top);
      den += f * pw[D + 1];
      num += f * pw[d];
    }
    const int hq = head_of(h), token = token_of(h);
    if (parts.splits == 1) {
      const __nv_bfloat16 v = __float2bfloat16_rn(den > 0.f ? num / den : den);        // (a sum that is not a number stays one)
      a.out[(size_t)token * a.out_stride + (size_t)hq * D + d] = *reinterpret_cast<const uint16_t*>(&v);
    } else if (joined) {
      sum[h * ROW + d] = num;
      if (d == 0) *reinterpret_cast<float2*>(sum + h * ROW + D) = make_float2(top, den);
    } else {
      const size_t ix = ((size_t)token * a.Hq + hq) * parts.splits + split;
      parts.o[ix * D + d] = num;
      if (d == 0) { parts.ml[ix * 2] = top; parts.ml[ix * 2 + 1] = den; }
    }
  }
  if (!joined) return;
  // ---- every CTA of the cluster joins a share of the heads' dims, all splits' partials in flight, in the order of the splits
  cluster_sync_all();
  for (int e = split * NW * 32 + threadIdx.x; e < heads * D; e += parts.splits * NW * 32) {
    const int h = e / D, d = e % D;
    float m[JOIN8], l[JOIN8], o[JOIN8], top = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
    for (int j = 0; j < JOIN8; ++j)
      if (j < parts.splits) {
        const uint32_t at = map_to_cta(smem_addr(sum + h * ROW), (uint32_t)j);
        m[j] = ld_cluster_f32(at + D * 4);
        l[j] = ld_cluster_f32(at + (D + 1) * 4);
        o[j] = ld_cluster_f32(at + d * 4);
      }
#pragma unroll
    for (int j = 0; j < JOIN8; ++j)
      if (j < parts.splits) top = fmaxf(top, m[j]);
#pragma unroll
    for (int j = 0; j < JOIN8; ++j)
      if (j < parts.splits && m[j] != -INFINITY) {                // (a split without tokens weighs nothing)
        const float f = ex2(m[j] - top);
        den += f * l[j];
        num += f * o[j];
      }
    const __nv_bfloat16 v = __float2bfloat16_rn(den > 0.f ? num / den : den);
    a.out[(size_t)token_of(h) * a.out_stride + (size_t)head_of(h) * D + d] = *reinterpret_cast<const uint16_t*>(&v);
  }
  cluster_sync_all();                                             // nobody leaves while a peer still reads its partials
}

// Weighs the split partials of a (token, query head) by exp2(m_j - max m) and normalises.  Latency bounds it: WPR warps share a row
// (four beyond four splits), lane j takes (m, l) of split j, a round's partials are all in flight.  The splits are added in an order
// of their own, whichever finished first.
constexpr int MERGE8 = 4;
template <int D, int WPR>
__global__ void __launch_bounds__(MERGE8 * 32) kv8_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                                const int* __restrict__ cu, int B, uint16_t* __restrict__ out,
                                                                long long out_stride, int Hq, int splits, long long rows) {
  constexpr int PL = D / 32;
  __shared__ float s_num[MERGE8][D];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
  const long long row = (long long)blockIdx.x * (MERGE8 / WPR) + warp / WPR;
  if (row >= rows) return;                                        // (WPR = 4: one row per CTA, never beyond)
  if (cu && (row / Hq < cu[0] || row / Hq >= cu[B])) return;      // rows of no sequence (the whole CTA with WPR = 4)
  const float* const ml = part_ml + row * splits * 2;
  if (ml[1] < 0.f) return;                                        // a row that was not split: its output stands already
  const float* const po = part_o + row * splits * D + PL * lane;
  float top = -INFINITY;
  for (int j = lane; j < splits; j += 32) top = fmaxf(top, ml[2 * j]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  float den = 0.f, num[PL];
#pragma unroll
  for (int d = 0; d < PL; ++d) num[d] = 0.f;
  for (int c = 0; c < splits; c += 32) {
    float m = -INFINITY, l = 0.f;
    if (c + lane < splits) { m = ml[2 * (c + lane)]; l = ml[2 * (c + lane) + 1]; }
    const float f = m == -INFINITY ? 0.f : exp2f(m - top);        // (a split without tokens weighs nothing)
    den += f * l;
    constexpr int U = WPR == 1 ? 4 : 8;
    for (int k0 = 0; k0 < 32 && c + k0 < splits; k0 += U * WPR) {
      float o[U][PL];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int j = c + k0 + sub + WPR * k;
#pragma unroll
        for (int d = 0; d < PL; d += 2) {
          const float2 v = j < splits ? *reinterpret_cast<const float2*>(po + (size_t)j * D + d) : make_float2(0.f, 0.f);
          o[k][d] = v.x;
          o[k][d + 1] = v.y;
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const float fj = __shfl_sync(FULL, f, k0 + sub + WPR * k);
#pragma unroll
        for (int d = 0; d < PL; ++d) num[d] += fj == 0.f ? 0.f : fj * o[k][d];
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) den += __shfl_xor_sync(FULL, den, o);
  if (WPR > 1) {
#pragma unroll
    for (int d = 0; d < PL; ++d) s_num[warp][PL * lane + d] = num[d];
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w)
#pragma unroll
      for (int d = 0; d < PL; ++d) num[d] += s_num[warp + w][PL * lane + d];
  }
  const float inv = den > 0.f ? 1.f / den : den;
  uint16_t* const at = out + row / Hq * out_stride + row % Hq * D + PL * lane;
#pragma unroll
  for (int d = 0; d < PL; d += 2) *reinterpret_cast<uint32_t*>(at + d) = pack_bf16(num[d] * inv, num[d + 1] * inv);
}

template <int D, int NW, int STG, bool CHUNK>
int attn8_launch(const Attn8& a, const Parts8& parts, long long ctas, cudaStream_t st_) {
  constexpr int smem = NW * STG * (2 * PAGE * D + 8 + 8);
  static std::atomic<uint64_t> set{0};                            // devices whose limit has been raised
  int dev = 0;
  if (int e = st::cuda_fail(cudaGetDevice(&dev), "st_kv8_attn: device")) return e;
  if (dev > 63 || !(set.load() >> dev & 1)) {
    if (int e = st::cuda_fail(cudaFuncSetAttribute(kv8_attn_kernel<D, NW, STG, CHUNK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                              "st_kv8_attn: shared memory attribute"))
      return e;
    if (dev <= 63) set.fetch_or(1ull << dev);
  }
  if (parts.splits == 1 || parts.o)
    return st::launch("st_kv8_attn launch", kv8_attn_kernel<D, NW, STG, CHUNK>, dim3((unsigned)ctas), dim3(NW * 32), (size_t)smem, st_,
                      a, parts, st::status_ptr());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(NW * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st_;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = st::pdl_enabled() ? 2 : 1;
  return st::cuda_fail(cudaLaunchKernelEx(&cfg, kv8_attn_kernel<D, NW, STG, CHUNK>, a, parts, st::status_ptr()), "st_kv8_attn launch");
}
// Do the splits of a unit join on chip, as a cluster?  Up to a wave of CTAs (us on chip / through memory and a second launch: 7 CTAs a unit,
// 1 x 1000 tokens 5.6 / 6.6; 64 CTAs, 1 x 4000 7.0 / 8.1; 256, 4 x 4000 9.5 / 10.7; 512, 16 x 4000 18.5 / 19.3, 8 x 16000 32.6 / 31.2),
// beyond it CTAs wait for their cluster's to find room (32 x 4000 with four splits 33.0 / 31.5, 64 x 8000 with eight 104 / 88).
bool joins8(long long ctas, int64_t splits) { return splits > 1 && splits <= JOIN8 && ctas <= 4ll * st::sm_count(); }
// An SM holds sixteen warps: four CTAs of four, or two of eight for a grid of at most two CTAs per SM (us with eight / four warps, 8 KV heads,
// lengths spread: 128 CTAs, 1 x 16K 10.7 / 13.4; 256, 4 x 16K 20.9 / 24.4; 512, 16 x 16K 61.1 / 57.5, 32 x 4K 33.7 / 30.6)
template <bool CHUNK>
int attn8_any(const char* who, const Attn8& a, const Parts8& given, int D, long long ctas, bool joined, cudaStream_t st_) {
  ST_REQUIRE(ctas < (1ll << 31), "%s: grid too large", who);
  Parts8 parts = given;
  if (joined) parts.o = parts.ml = nullptr;
  const bool wide = ctas <= 2ll * st::sm_count();
  int e;
  if (D == 128) e = wide ? attn8_launch<128, 8, 3, CHUNK>(a, parts, ctas, st_) : attn8_launch<128, 4, 3, CHUNK>(a, parts, ctas, st_);
  else e = wide ? attn8_launch<64, 8, 5, CHUNK>(a, parts, ctas, st_) : attn8_launch<64, 4, 5, CHUNK>(a, parts, ctas, st_);
  return e || joined || parts.splits == 1 ? e : merge8(who, a, parts, D, st_);
}
long long decode_ctas(int64_t B, int64_t Hq, int64_t Hkv, int64_t S) { return B * Hkv * ((Hq / Hkv + 7) / 8) * S; }
bool decode_joins(int64_t B, int64_t Hq, int64_t Hkv, int64_t S) { return joins8(decode_ctas(B, Hq, Hkv, S), S); }
// (the grid has room for a part-filled tile of every sequence; about as many as the rows or the sequences need find work)
bool rows8_joins(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t S) {
  return joins8(std::max(B, (T * (Hq / Hkv) + 7) / 8) * Hkv * S, S);
}
}  // namespace

namespace st {
int rows8_attn(const char* who, const Attn8& a, const Parts8& parts, int D, cudaStream_t st_) {
  const long long slots = a.T * (a.Hq / a.H) / 8 + a.B;
  return attn8_any<true>(who, a, parts, D, slots * a.H * parts.splits, rows8_joins(a.T, a.B, a.Hq, a.H, parts.splits), st_);
}
int merge8(const char* who, const Attn8& a, const Parts8& parts, int D, cudaStream_t st_) {
  const long long rows = a.T * a.Hq;
  const int per_cta = parts.splits > 4 ? 1 : MERGE8;
  auto* kernel = D == 128 ? (parts.splits > 4 ? kv8_merge_kernel<128, MERGE8> : kv8_merge_kernel<128, 1>)
                          : (parts.splits > 4 ? kv8_merge_kernel<64, MERGE8> : kv8_merge_kernel<64, 1>);
  return st::launch(who, kernel, dim3((unsigned)((rows + per_cta - 1) / per_cta)), dim3(MERGE8 * 32), 0, st_, (const float*)parts.o,
                    (const float*)parts.ml, a.cu, a.B, a.out, a.out_stride, a.Hq, parts.splits, rows);
}
}  // namespace st

extern "C" int64_t st_kv8_page_bytes(int64_t H, int64_t D) { return H * 2 * st::PAGE * D; }

extern "C" int st_kv8_append(const void* K, const void* V, int64_t ks, int64_t vs, const int64_t* slot, int64_t N, int64_t H,
                             int64_t D, void* kv, int8_t* exps, int64_t nblocks, const int64_t* pos, int64_t pos_step,
                             const float* cos_t, const float* sin_t, int64_t max_pos, int interleaved, const void* wk, const void* Q,
                             int64_t qs, const void* wq, int64_t Hq, void* q_out, int64_t qos, double eps, int32_t* marks,
                             int32_t* bad, void* stream) {
  ST_REQUIRE(N >= 0 && H > 0 && nblocks >= 0, "st_kv8_append: negative size");
  ST_REQUIRE(D == 64 || D == 128, "st_kv8_append: head dimension 64 or 128 (got %lld)", (long long)D);
  if (N == 0) return 0;
  ST_REQUIRE(K && V && slot && kv && exps && bad, "st_kv8_append: null pointer");
  ST_REQUIRE(ks % 8 == 0 && vs % 8 == 0 && ks >= 0 && vs >= 0 && st::aligned16(K) && st::aligned16(V) && st::aligned16(kv),
             "st_kv8_append: K / V must be 16-byte aligned [N, H, D] with heads contiguous and token strides that are multiples of 8");
  ST_REQUIRE((cos_t == nullptr) == (sin_t == nullptr) && (cos_t == nullptr || (pos && max_pos > 0)),
             "st_kv8_append: a rotation takes positions and both tables");
  ST_REQUIRE(st::aligned16(cos_t) && st::aligned16(sin_t) && st::aligned16(wk) && st::aligned16(wq), "st_kv8_append: tables and norm weights must be 16-byte aligned");
  ST_REQUIRE(pos_step == 0 || pos_step == 1, "st_kv8_append: pos_step is 1, or 0 for one position of all tokens");
  ST_REQUIRE(Q == nullptr || (q_out && Hq > 0 && qs % 8 == 0 && qos % 8 == 0 && qs >= 0 && qos >= 0 && st::aligned16(Q) && st::aligned16(q_out)),
             "st_kv8_append: queries and their output must be 16-byte aligned with token strides that are multiples of 8");
  ST_REQUIRE(Q == nullptr || N == 1 || qos >= Hq * D, "st_kv8_append: rows of the queries' output overlap");
  const bool scan = N <= SCAN_MAX;
  ST_REQUIRE(scan || marks, "st_kv8_append: calls of more than %d tokens need marks (int32 [17 * blocks], zero)", SCAN_MAX);
  ST_REQUIRE(N < (1ll << 31) - 16 && N * H < (1ll << 32) && (Q == nullptr || N * Hq < (1ll << 34)), "st_kv8_append: too large");
  Append8 a;
  a.K = (const uint16_t*)K; a.V = (const uint16_t*)V; a.Q = (const uint16_t*)Q;
  a.ks = ks; a.vs = vs; a.qs = qs; a.qos = qos; a.slot = (const long long*)slot;
  a.kv = (uint8_t*)kv; a.exps = exps; a.nblocks = nblocks;
  a.pos = (const long long*)pos; a.pos_step = pos_step; a.max_pos = max_pos; a.cos_t = cos_t; a.sin_t = sin_t;
  a.wq = (const uint16_t*)wq; a.wk = (const uint16_t*)wk; a.q_out = (uint16_t*)q_out; a.marks = marks; a.bad = bad;
  a.N = (int)N; a.H = (int)H; a.Hq = Q ? (int)Hq : 0; a.eps = (float)eps; a.pairs = interleaved ? 1 : 0;
  const cudaStream_t st_ = (cudaStream_t)stream;
  a.run = (int)std::min<long long>(st::PAGE, std::max<long long>(1, N / (8ll * st::sm_count())));
  const long long page_ctas = scan ? (N * H * 2 + 7) / 8 : (N + a.run - 1) / a.run;
  // queries: a warp per group of heads while that leaves SMs without one, else up to eight groups of a token (the whole append, us with
  // one / eight groups: 16 sequences 4.6 / 5.0, 2048 tokens of one 18.5 / 16.9, 4096 35.3 / 24.7)
  const int groups = (int)((a.Hq + 512 / D - 1) / (512 / D));
  a.q_steps = (int)std::min<long long>(std::min(std::max(groups, 1), 8), std::max<long long>(1, N * groups / (16ll * st::sm_count())));
  a.q_units = groups ? (groups + a.q_steps - 1) / a.q_steps : 0;
  const long long q_ctas = (N * a.q_units + 7) / 8;
  ST_REQUIRE(page_ctas + q_ctas < (1ll << 31), "st_kv8_append: too large");
  a.q_cta = (int)page_ctas;
  if (!scan)
    if (int e = st::launch("st_kv8_append marks", kv8_mark_kernel, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, st_, a)) return e;
  auto* kernel = D == 128 ? (scan ? kv8_append_kernel<128, true> : kv8_append_kernel<128, false>)
                          : (scan ? kv8_append_kernel<64, true> : kv8_append_kernel<64, false>);
  return st::launch("st_kv8_append launch", kernel, dim3((unsigned)(page_ctas + q_ctas)), dim3(256), 0, st_, a);
}

extern "C" int st_kv8_dequant_blocks(const void* kv, const int8_t* exps, int64_t nblocks, int64_t H, int64_t D, const int32_t* blocks,
                                     int64_t n, void* Kd, void* Vd, void* stream) {
  ST_REQUIRE(n >= 0 && H > 0 && nblocks >= 0, "st_kv8_dequant_blocks: negative size");
  ST_REQUIRE(D == 64 || D == 128, "st_kv8_dequant_blocks: head dimension 64 or 128 (got %lld)", (long long)D);
  if (n == 0) return 0;
  ST_REQUIRE(kv && exps && Kd && Vd, "st_kv8_dequant_blocks: null pointer");
  ST_REQUIRE(blocks || n <= nblocks, "st_kv8_dequant_blocks: more pages than there are");
  ST_REQUIRE(st::aligned16(kv) && st::aligned16(Kd) && st::aligned16(Vd), "st_kv8_dequant_blocks: alignment");
  const long long threads = n * H * 2 * (st::PAGE * D / 16);
  ST_REQUIRE((threads + 255) / 256 < (1ll << 31), "st_kv8_dequant_blocks: too large");
  auto* kernel = D == 128 ? kv8_dequant_kernel<128> : kv8_dequant_kernel<64>;
  return st::launch("st_kv8_dequant launch", kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, (cudaStream_t)stream,
                    (const uint8_t*)kv, exps, (long long)nblocks, (int)H, (const int*)blocks, (long long)n, (uint16_t*)Kd, (uint16_t*)Vd);
}

namespace st {
// what both forms of the attention check and pass on
int attn8_args(Attn8& a, const char* who, const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv,
               const int8_t* exps, int64_t nblocks, int64_t Hkv, int64_t D, const int32_t* bt, int64_t btw, int64_t bts, const int32_t* lens,
               const int32_t* starts, int64_t window, void* out, int64_t os, double scale) {
  ST_REQUIRE(T >= 0 && B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "%s: heads", who);
  ST_REQUIRE(D == 64 || D == 128, "%s: head dimension 64 or 128 (got %lld)", who, (long long)D);
  ST_REQUIRE(scale > 0 && scale <= 512, "%s: the softmax scale must be positive and at most 512", who);
  ST_REQUIRE(window >= 0 && window < (1ll << 31), "%s: window", who);
  if (T == 0 || B == 0) return 0;
  ST_REQUIRE(q && kv && exps && bt && lens && out, "%s: null pointer", who);
  ST_REQUIRE(nblocks > 0 && btw > 0 && bts >= 0, "%s: empty cache or block table", who);
  ST_REQUIRE(st::aligned16(q) && st::aligned16(out) && st::aligned16(kv) && qs % 8 == 0 && os % 8 == 0 && qs >= 0 && os >= 0,
             "%s: q, out and the pages must be 16-byte aligned, token strides multiples of 8", who);
  ST_REQUIRE(((uintptr_t)exps & 1u) == 0, "%s: exponents must be 2-byte aligned", who);
  ST_REQUIRE(T == 1 || os >= Hq * D, "%s: rows of out overlap", who);
  ST_REQUIRE(T * Hq < (1ll << 31) && btw < (1ll << 27), "%s: too large", who);
  a.q = (const uint16_t*)q; a.q_stride = qs; a.cu = cu; a.kv = (const uint8_t*)kv; a.exps = exps; a.nblocks = nblocks;
  a.table = bt; a.table_stride = bts; a.table_width = (int)btw; a.lens = lens; a.starts = starts; a.out = (uint16_t*)out; a.out_stride = os;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.B = (int)B; a.Hq = (int)Hq; a.H = (int)Hkv; a.window = (int)window; a.T = T;
  return 0;
}
}  // namespace st

extern "C" int st_kv8_attn(const void* q, int64_t qs, int64_t B, int64_t Hq, const void* kv, const int8_t* exps, int64_t nblocks,
                           int64_t Hkv, int64_t D, const int32_t* bt, int64_t bts, const int32_t* lens, const int32_t* starts,
                           int64_t window, void* out, int64_t os, float* wo, float* wml, double scale, int64_t S, int64_t minpps,
                           void* stream) {
  return st_kv8_attn_table(q, qs, B, Hq, kv, exps, nblocks, Hkv, D, bt, bts, bts, lens, starts, window, out, os, wo, wml, scale, S, minpps, stream);
}

extern "C" int st_kv8_attn_table(const void* q, int64_t qs, int64_t B, int64_t Hq, const void* kv, const int8_t* exps, int64_t nblocks,
                                 int64_t Hkv, int64_t D, const int32_t* bt, int64_t btw, int64_t bts, const int32_t* lens,
                                 const int32_t* starts, int64_t window, void* out, int64_t os, float* wo, float* wml, double scale,
                                 int64_t S, int64_t minpps, void* stream) {
  Attn8 a;
  if (int e = attn8_args(a, "st_kv8_attn", q, qs, B, Hq, nullptr, B, kv, exps, nblocks, Hkv, D, bt, btw, bts, lens, starts, window, out, os,
                         scale))
    return e;
  ST_REQUIRE(S >= 1 && S <= 1024, "st_kv8_attn: splits must be in [1, 1024]");
  ST_REQUIRE((wo && wml && st::aligned16(wo)) || st_kv8_attn_workspace_bytes(B, B, Hq, Hkv, D, S, 0) == 0,
             "st_kv8_attn: split workspace (wo, wml) missing or unaligned");
  if (B == 0) return 0;
  ST_REQUIRE(st::status_ptr() != nullptr, "st_kv8_attn: no device status word");
  const Parts8 parts = {wo, wml, (int)S, (int)(minpps < 1 ? 1 : minpps)};
  const cudaStream_t st_ = (cudaStream_t)stream;
  return attn8_any<false>("st_kv8_attn", a, parts, (int)D, decode_ctas(B, Hq, Hkv, S), decode_joins(B, Hq, Hkv, S), st_);
}

extern "C" int64_t st_kv8_attn_workspace_bytes(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t S, int chunk) {
  if (T <= 0 || B <= 0 || Hkv <= 0 || S <= 1) return 0;
  if (!chunk ? decode_joins(B, Hq, Hkv, S) : few_rows8(T, B, Hq / Hkv) && rows8_joins(T, B, Hq, Hkv, S)) return 0;
  return T * Hq * S * (D + 2) * 4;
}
