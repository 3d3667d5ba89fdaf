// KV pages in 8 bits on sm_100a: append (rotation and quantisation on the way), read-back, and attention over the pages.
// The page and why it is laid out so: st_kv8.cuh.
#include <math.h>

#include "../../include/statetree_b200.h"
#include "st_host.h"
#include "st_kv8.cuh"

namespace {
using namespace st;

// ------------------------------------------------------------------------------------------------ append
// Keys (normalised and rotated on the way, in fp32, one rounding to e4m3 at the end), values, and the queries of the same tokens
// (normalised and rotated into q_out).  A warp owns one unit (page, head, K or V) for the launch and takes every token of the call
// that goes to the page, so nothing is added or compared between warps and the result does not depend on their order:
//     e' = the smallest exponent that holds the new rows; the page's old one if that is larger and the page does not start anew
//     new rows are rounded at e', the others again at e' if it differs from the old exponent, or cleared if row 0 is among the new
// Which warp: the last token of the call in a page leads it.
//   SCAN  (calls of up to SCAN_MAX tokens) a warp per (token, unit) walks the call's slots and finds out itself
//   else  kv8_mark_kernel leaves every row's and page's last token in `marks`; a CTA takes sixteen tokens of the call, all units of
//         the pages they lead, and clears what it read
// Same slot twice: the last one counts in both.  Values that are not finite are stored as the largest of their sign (infinities) or
// as zero (NaN), and flagged in *bad.
constexpr int SCAN_MAX = 512;

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
  int N, H, Hq, q_cta;                             // q_cta: first CTA that works on queries
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
__device__ __forceinline__ void row_norm(float (&f)[16], const uint16_t* w, float eps, int c) {
  constexpr int LPR = D / 16;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
  const float r = __frsqrt_rn(ss * (1.f / D) + eps);
  float g[16];
  unpack8(*reinterpret_cast<const uint4*>(w + 8 * c), g, 0);
  unpack8(*reinterpret_cast<const uint4*>(w + D / 2 + 8 * c), g, 8);
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = f[i] * r * g[i];
}
template <int D>
__device__ __forceinline__ void row_rotate(float (&f)[16], const float* ct, const float* st, int pairs, int c) {
  float cs[8], sn[8];
  const int p0 = pairs ? 4 * c : 8 * c, p1 = pairs ? D / 4 + 4 * c : 8 * c + 4;
  *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(ct + p0);
  *reinterpret_cast<float4*>(cs + 4) = *reinterpret_cast<const float4*>(ct + p1);
  *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(st + p0);
  *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(st + p1);
  if (pairs) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {                  // pair i of the lane: f[2i], f[2i + 1]
      const float a = f[2 * i], b = f[2 * i + 1];
      f[2 * i] = a * cs[i] - b * sn[i];
      f[2 * i + 1] = a * sn[i] + b * cs[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = f[i], b = f[8 + i];
      f[i] = a * cs[i] - b * sn[i];
      f[8 + i] = a * sn[i] + b * cs[i];
    }
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

// one unit: lane r < 16 holds in `tok` the token that goes to row r, -1 = none; at least one row has a token
template <int D>
__device__ __forceinline__ void append_unit(const Append8& a, long long page, int h, int kvi, int tok, int lane) {
  constexpr int LPR = D / 16, RPI = 32 / LPR, ITER = PAGE / RPI;
  const unsigned rows = __ballot_sync(FULL, lane < PAGE && tok >= 0);
  const int c = lane % LPR;
  const uint16_t* const src = (kvi ? a.V : a.K) + (size_t)h * D + 8 * c;
  const long long step = kvi ? a.vs : a.ks;
  uint4 raw[ITER][2];
  int mine[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    mine[i] = __shfl_sync(FULL, tok, i * RPI + lane / LPR);
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
  float f[ITER][16], top = 0.f;
  bool odd = false;                                // (a value that is not finite)
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    unpack8(raw[i][0], f[i], 0);
    unpack8(raw[i][1], f[i], 8);
    if (kvi == 0) {
      if (a.wk) row_norm<D>(f[i], a.wk, a.eps, c);
      if (a.cos_t && mine[i] >= 0) {
        const long long at = table_row(a, mine[i]) * (D / 2);
        row_rotate<D>(f[i], a.cos_t + at, a.sin_t + at, a.pairs, c);
      }
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float m = fabsf(f[i][k]);
      const bool fin = m < INFINITY;
      odd |= !fin;
      top = fmaxf(top, fin ? m : 0.f);
      if (m != m) f[i][k] = 0.f;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  const int e = max(was, exp_for(top));
  // (a finite value beyond 448 * 2^E8_MAX is cut off there, as infinities are)
  odd |= top > 448.f * pow2i(E8_MAX);
  const float down = pow2i(-e), up = pow2i(20 + was);
  uint8_t* const unit = a.kv + page8_off<D>(page, a.H, h, kvi);
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int r = i * RPI + lane / LPR;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int d = half * (D / 2) + 8 * c;
      uint2* const at = reinterpret_cast<uint2*>(unit + r * D + 16 * piece8<D>(r, d >> 4) + (d & 8));
      if (mine[i] >= 0) *at = e4m3_eight(f[i] + 8 * half, down);
      else if (anew) *at = make_uint2(0, 0);
      else if (e != was) *at = rescale_eight(*at, up, down);
    }
  }
  __syncwarp();                                    // (every lane has read the old exponent)
  if (lane == 0 && (anew || e != was)) *exp_at = (int8_t)e;
  if (odd) *a.bad = 1;
}

// rows [first, ..) of the queries [N * Hq, D]: a warp takes 32 / (D / 16) of them
template <int D>
__device__ __forceinline__ void rotate_queries(const Append8& a, long long first, int lane) {
  constexpr int LPR = D / 16;
  const long long row = first + lane / LPR;
  const bool live = row < (long long)a.N * a.Hq;
  const long long token = live ? row / a.Hq : 0;
  const int h = live ? (int)(row % a.Hq) : 0, c = lane % LPR;
  const uint16_t* const p = a.Q + token * a.qs + (size_t)h * D + 8 * c;
  float f[16];
  unpack8(*reinterpret_cast<const uint4*>(p), f, 0);
  unpack8(*reinterpret_cast<const uint4*>(p + D / 2), f, 8);
  if (a.wq) row_norm<D>(f, a.wq, a.eps, c);
  if (a.cos_t) {
    const long long at = table_row(a, token) * (D / 2);
    row_rotate<D>(f, a.cos_t + at, a.sin_t + at, a.pairs, c);
  }
  if (!live) return;
  uint16_t* const o = a.q_out + token * a.qos + (size_t)h * D + 8 * c;
  *reinterpret_cast<uint4*>(o) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  *reinterpret_cast<uint4*>(o + D / 2) =
      make_uint4(pack_bf16(f[8], f[9]), pack_bf16(f[10], f[11]), pack_bf16(f[12], f[13]), pack_bf16(f[14], f[15]));
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
__global__ void __launch_bounds__(256) kv8_append_kernel(const Append8 a) {
  __shared__ int s_row[8][PAGE];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, units = 2 * a.H;
  if ((int)blockIdx.x >= a.q_cta) {
    const long long first = ((long long)((int)blockIdx.x - a.q_cta) * 8 + warp) * (512 / D);
    if (first < (long long)a.N * a.Hq) rotate_queries<D>(a, first, lane);
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
    append_unit<D>(a, page, u >> 1, u & 1, lane < PAGE ? row[lane] : -1, lane);
  } else {
    const int i = (int)blockIdx.x * PAGE + lane;
    const long long s = lane < PAGE && i < a.N ? a.slot[i] : -1;
    const bool leads = slot_ok(a, s) && a.marks[a.nblocks * PAGE + s / PAGE] == i + 1;
    unsigned left = __ballot_sync(FULL, leads);    // (the same in every warp: a mark of this CTA's pages is cleared below, behind a barrier)
    const unsigned all = left;
    for (; left; left &= left - 1) {
      const long long page = __shfl_sync(FULL, s, __ffs(left) - 1) / PAGE;
      const int tok = lane < PAGE ? a.marks[page * PAGE + lane] - 1 : -1;
      for (int u = warp; u < units; u += 8) append_unit<D>(a, page, u >> 1, u & 1, tok, lane);
    }
    __syncthreads();
    if (warp == 0)
      for (left = all; left; left &= left - 1) {
        const long long page = __shfl_sync(FULL, s, __ffs(left) - 1) / PAGE;
        if (lane < PAGE) a.marks[page * PAGE + lane] = 0;
        if (lane == PAGE) a.marks[a.nblocks * PAGE + page] = 0;
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

// ------------------------------------------------------------------------------------------------ attention, plain
// One warp per (query token, head); keys one after the other, the running maximum and sum of the softmax in fp32.
struct Attn8 {
  const uint16_t* q; long long q_stride;
  const int* cu;                                   // first query of each sequence [B + 1]; nullptr: one query each
  const uint8_t* kv; const int8_t* exps; long long nblocks;
  const int* table; long long table_stride;
  const int* lens; const int* starts;
  uint16_t* out; long long out_stride;
  float scale_log2;
  int B, Hq, H, window;
  long long T;
};
template <int D>
__global__ void __launch_bounds__(256) kv8_rows_kernel(const Attn8 a) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int PL = D / 32;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long t = w / a.Hq;
  if (t >= a.T) return;
  const int hq = (int)(w % a.Hq), h = hq / (a.Hq / a.H);
  int b = (int)t, n = 1, i = 0;
  if (a.cu) {
    for (b = 0; b < a.B && a.cu[b + 1] <= t; ++b) {}
    if (b >= a.B || t < a.cu[b]) return;
    n = a.cu[b + 1] - a.cu[b];
    i = (int)t - a.cu[b];
  }
  const int pos = a.lens[b] - n + i, end = (int)min((long long)pos, a.table_stride * PAGE - 1);
  int lo = a.starts ? max(a.starts[b], 0) : 0;
  if (a.window > 0) lo = max(lo, pos - a.window + 1);
  float q[PL], o[PL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < PL; ++k) {
    q[k] = __uint_as_float((uint32_t)a.q[t * a.q_stride + (size_t)hq * D + PL * lane + k] << 16);
    o[k] = 0.f;
  }
  for (int j = lo; j <= end; ++j) {
    long long blk = a.table[b * a.table_stride + j / PAGE];
    blk = blk < 0 ? 0 : (blk >= a.nblocks ? a.nblocks - 1 : blk);
    const int r = j % PAGE, at = r * D + 16 * piece8<D>(r, PL * lane >> 4) + (PL * lane & 15);
    float k[PL], v[PL];
#pragma unroll
    for (int kvi = 0; kvi < 2; ++kvi) {
      const float up = pow2i(20 + page8_exp(a.exps[((size_t)blk * a.H + h) * 2 + kvi]));
      const uint8_t* p = a.kv + page8_off<D>(blk, a.H, h, kvi) + at;
#pragma unroll
      for (int d = 0; d < PL; d += 2) {
        uint32_t p01, p23;
        codes_to_bf16((uint32_t)p[d] | (uint32_t)p[d + 1] << 8, p01, p23);
        const float2 x = codes_value(p01, up);
        (kvi ? v : k)[d] = x.x;
        (kvi ? v : k)[d + 1] = x.y;
      }
    }
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < PL; ++d) s = fmaf(q[d], k[d], s);
#pragma unroll
    for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(FULL, s, off);
    s *= a.scale_log2;
    const float top = fmaxf(m, s), f = exp2f(m - top), p = exp2f(s - top);
    l = l * f + p;
#pragma unroll
    for (int d = 0; d < PL; ++d) o[d] = o[d] * f + p * v[d];
    m = top;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int d = 0; d < PL; d += 2)
    *reinterpret_cast<uint32_t*>(a.out + t * a.out_stride + (size_t)hq * D + PL * lane + d) = pack_bf16(o[d] * inv, o[d + 1] * inv);
}
}  // namespace

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
  const long long page_ctas = scan ? (N * H * 2 + 7) / 8 : (N + st::PAGE - 1) / st::PAGE;
  const long long per_cta = 8 * 512 / D, q_ctas = (N * a.Hq + per_cta - 1) / per_cta;
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

namespace {
// what both forms of the attention check and pass on
int attn8_args(Attn8& a, const char* who, const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv,
               const int8_t* exps, int64_t nblocks, int64_t Hkv, int64_t D, const int32_t* bt, int64_t bts, const int32_t* lens,
               const int32_t* starts, int64_t window, void* out, int64_t os, double scale) {
  ST_REQUIRE(T >= 0 && B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "%s: heads", who);
  ST_REQUIRE(D == 64 || D == 128, "%s: head dimension 64 or 128 (got %lld)", who, (long long)D);
  ST_REQUIRE(scale > 0 && scale <= 512, "%s: the softmax scale must be positive and at most 512", who);
  ST_REQUIRE(window >= 0 && window < (1ll << 31), "%s: window", who);
  if (T == 0 || B == 0) return 0;
  ST_REQUIRE(q && kv && exps && bt && lens && out, "%s: null pointer", who);
  ST_REQUIRE(nblocks > 0 && bts > 0, "%s: empty cache or block table", who);
  ST_REQUIRE(st::aligned16(q) && st::aligned16(out) && st::aligned16(kv) && qs % 8 == 0 && os % 8 == 0 && qs >= 0 && os >= 0,
             "%s: q, out and the pages must be 16-byte aligned, token strides multiples of 8", who);
  ST_REQUIRE(T * Hq < (1ll << 31) && bts < (1ll << 27), "%s: too large", who);
  a.q = (const uint16_t*)q; a.q_stride = qs; a.cu = cu; a.kv = (const uint8_t*)kv; a.exps = exps; a.nblocks = nblocks;
  a.table = bt; a.table_stride = bts; a.lens = lens; a.starts = starts; a.out = (uint16_t*)out; a.out_stride = os;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.B = (int)B; a.Hq = (int)Hq; a.H = (int)Hkv; a.window = (int)window; a.T = T;
  return 0;
}
}  // namespace

extern "C" int st_kv8_attn(const void* q, int64_t qs, int64_t B, int64_t Hq, const void* kv, const int8_t* exps, int64_t nblocks,
                           int64_t Hkv, int64_t D, const int32_t* bt, int64_t bts, const int32_t* lens, const int32_t* starts,
                           int64_t window, void* out, int64_t os, float* wo, float* wml, double scale, int64_t S, int64_t minpps,
                           void* stream) {
  Attn8 a;
  if (int e = attn8_args(a, "st_kv8_attn", q, qs, B, Hq, nullptr, B, kv, exps, nblocks, Hkv, D, bt, bts, lens, starts, window, out, os, scale))
    return e;
  ST_REQUIRE(S >= 1 && S <= 1024, "st_kv8_attn: splits must be in [1, 1024]");
  ST_REQUIRE(S == 1 || (wo && wml && st::aligned16(wo)), "st_kv8_attn: split workspace (wo, wml) missing or unaligned");
  if (B == 0) return 0;
  return st::launch("st_kv8_attn launch", D == 128 ? kv8_rows_kernel<128> : kv8_rows_kernel<64>, dim3((unsigned)((B * Hq + 7) / 8)), dim3(256),
                    0, (cudaStream_t)stream, a);
}

extern "C" int st_kv8_chunk_attn(const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv,
                                 const int8_t* exps, int64_t nblocks, int64_t Hkv, int64_t D, const int32_t* bt, int64_t bts,
                                 const int32_t* lens, const int32_t* starts, int64_t window, void* out, int64_t os, float* wo,
                                 float* wml, double scale, int64_t S, void* stream) {
  Attn8 a;
  if (int e = attn8_args(a, "st_kv8_chunk_attn", q, qs, T, Hq, cu, B, kv, exps, nblocks, Hkv, D, bt, bts, lens, starts, window, out, os, scale))
    return e;
  ST_REQUIRE(S >= 1 && S <= 1024, "st_kv8_chunk_attn: splits must be in [1, 1024]");
  ST_REQUIRE(S == 1 || (wo && wml && st::aligned16(wo)), "st_kv8_chunk_attn: split workspace (wo, wml) missing or unaligned");
  if (T == 0 || B == 0) return 0;
  ST_REQUIRE(cu || T == B, "st_kv8_chunk_attn: without cu every sequence has one query");
  return st::launch("st_kv8_chunk_attn launch", D == 128 ? kv8_rows_kernel<128> : kv8_rows_kernel<64>, dim3((unsigned)((T * Hq + 7) / 8)),
                    dim3(256), 0, (cudaStream_t)stream, a);
}
