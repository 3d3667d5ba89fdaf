// Rotary positions of queries and keys: every pair (a, b) of a head's rotated part becomes (a c - b s, a s + b c) with the cosine and
// sine of its token's position, optionally behind a per-head RMSNorm.  The pairs are neighbours (2i, 2i + 1) or lie half of the part
// apart; values outside the part pass through.  With the sign of s turned the same kernel is the gradient (the transposed matrix).
//
// Bound by HBM: every value is read once and written once.  A lane owns VEC pairs (two 16-byte vectors) of a head, so that a pair
// never crosses lanes in either layout and the norm needs one reduction over the head's lanes; a warp walks the heads of ONE token, whose
// cosines and sines stay in registers.  Few tokens: the heads of a token are dealt to several warps.
// Measured, us in a graph (BF16, heads of 128): 32764 tokens of 32 + 8 heads 111 = 6.1 TB/s (a copy of as many bytes 105), with norms 118;
// 8190 tokens of 16 + 16 heads 26.8 (copy 24.7); 1261 tokens of 64 heads of 80, 32 of them rotated, 8.9; one token 2.9.  Two heads in flight
// and 24 warps an SM; with norms, whose arithmetic fills 70 % of the issue slots (two pairs an instruction: one 121), one and 32
// (two and 24: 130; the weights in registers 143; four in flight and 16 warps 159).
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/statetree_b200.h"
#include "st_common.cuh"
#include "st_host.h"

namespace {
using namespace st;

struct Side { const void* x; void* y; const void* w; long long xt, xh, yt, yh; int heads; };      // strides: tokens, heads
struct RotArgs {
  Side s[2];                                       // queries, keys
  const long long* pos; int pos_step;
  const float* cos_t; const float* sin_t; long long span;
  long long N;
  int D, part, offset, parts, lanes;               // parts: warps that share a token; lanes of a head (a power of two)
  float eps, sign;
};

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes as floats, and back
template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, float>) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, float>) {
      w[i] = __float_as_uint(f[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      w[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
    } else {
      const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ long long place(const RotArgs& a, long long n) {
  const long long p = a.pos[a.pos_step ? n : 0];
  return p < 0 ? 0 : (p >= a.span ? a.span - 1 : p);
}

constexpr int THREADS = 256;

template <typename T, bool PAIRS, bool NORM>
__global__ void __launch_bounds__(THREADS, NORM ? 4 : 3) rotate_kernel(const RotArgs a) {
  constexpr int VEC = 16 / sizeof(T);              // pairs of a lane = values of one of its two vectors
  constexpr int U = NORM ? 1 : 2;                  // heads whose loads are in flight together
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  const long long n = w / a.parts;
  pdl_wait();
  pdl_launch_dependents();
  if (n >= a.N) return;
  const int part = (int)(w % a.parts), li = lane & (a.lanes - 1), per = 32 / a.lanes;
  const int total = a.s[0].heads + a.s[1].heads, passes = (total + per - 1) / per;
  const int p0 = (int)((long long)passes * part / a.parts), p1 = (int)((long long)passes * (part + 1) / a.parts);
  // this lane's two vectors of every head
  const int s0 = li * VEC, half = a.part / 2;
  const float inv_d = 1.f / (float)a.D;
  const bool here = 2 * s0 < a.D, rot = s0 < half;
  int d0, d1;
  if (rot) {
    d0 = a.offset + (PAIRS ? 2 * s0 : s0);
    d1 = PAIRS ? d0 + VEC : d0 + half;
  } else {
    d0 = 2 * (s0 - half);
    d1 = d0 + VEC;
    d0 += d0 < a.offset ? 0 : a.part;
    d1 += d1 < a.offset ? 0 : a.part;
  }
  const bool second = here && d1 < a.D;            // (a rest of an odd number of vectors)
  auto head_of = [&](int p, int& kv) {             // head p * per + lane / lanes, -1 = none
    int h = p * per + lane / a.lanes;
    kv = h >= a.s[0].heads;
    h -= kv ? a.s[0].heads : 0;
    return p < p1 && h < a.s[kv].heads && here ? h : -1;
  };
  uint4 u[U][2];
  auto load = [&](int p, uint4 (&v)[2]) {
    int kv;
    const int h = head_of(p, kv);
    v[0] = v[1] = make_uint4(0, 0, 0, 0);
    if (h < 0) return;
    const T* const x = reinterpret_cast<const T*>(a.s[kv].x) + n * a.s[kv].xt + h * a.s[kv].xh;
    v[0] = *reinterpret_cast<const uint4*>(x + d0);
    if (second) v[1] = *reinterpret_cast<const uint4*>(x + d1);
  };
#pragma unroll
  for (int i = 0; i < U; ++i) load(p0 + i, u[i]);
  uint64_t c[VEC / 2], s[VEC / 2];                 // of two pairs each: cosines, sines
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) { c[i] = pair2(1.f, 1.f); s[i] = 0; }
  if (rot && here) {
    const long long row = place(a, n) * half + s0;
#pragma unroll
    for (int i = 0; i < VEC / 2; i += 2) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(a.cos_t + row + 2 * i)), y = __ldg(reinterpret_cast<const float4*>(a.sin_t + row + 2 * i));
      c[i] = pair2(x.x, x.y); c[i + 1] = pair2(x.z, x.w);
      s[i] = pair2(a.sign * y.x, a.sign * y.y); s[i + 1] = pair2(a.sign * y.z, a.sign * y.w);
    }
  }
  for (int p = p0; p < p1; p += U) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float f[2 * VEC];
      unpack<T>(u[i][0], f);
      unpack<T>(u[i][1], f + VEC);
      // pair k is (f[2k], f[2k + 1]) or (f[k], f[VEC + k]); two pairs at a time
      auto first = [](int k) { return PAIRS ? 2 * k : k; };
      auto other = [](int k) { return PAIRS ? 2 * k + 1 : VEC + k; };
      uint64_t x[VEC / 2], y2[VEC / 2];
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        x[k] = pair2(f[first(2 * k)], f[first(2 * k + 1)]);
        y2[k] = pair2(f[other(2 * k)], f[other(2 * k + 1)]);
      }
      int kv;
      const int h = head_of(p + i, kv);
      load(p + i + U, u[i]);
      if constexpr (NORM) {
        uint64_t sq = 0;
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) sq = fma2(y2[k], y2[k], fma2(x[k], x[k], sq));
        float q0, q1;
        unpair2(sq, q0, q1);
        float ss = q0 + q1;
        for (int o = a.lanes >> 1; o; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
        const T* const wt = reinterpret_cast<const T*>(a.s[kv].w);
        if (h >= 0 && wt) {                        // (from L1: held in registers they cost a quarter of the resident warps)
          const float r = rsqrtf(ss * inv_d + a.eps);
          const uint64_t r2 = pair2(r, r);
          float g[2 * VEC];
          unpack<T>(__ldg(reinterpret_cast<const uint4*>(wt + d0)), g);
          unpack<T>(second ? __ldg(reinterpret_cast<const uint4*>(wt + d1)) : make_uint4(0, 0, 0, 0), g + VEC);
#pragma unroll
          for (int k = 0; k < VEC / 2; ++k) {
            x[k] = mul2f(mul2f(x[k], r2), pair2(g[first(2 * k)], g[first(2 * k + 1)]));
            y2[k] = mul2f(mul2f(y2[k], r2), pair2(g[other(2 * k)], g[other(2 * k + 1)]));
          }
        }
      }
      if (h < 0) continue;
      if (rot) {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          const uint64_t t = fma2(x[k], c[k], mul2f(y2[k], s[k]) ^ 0x8000000080000000ull);
          y2[k] = fma2(x[k], s[k], mul2f(y2[k], c[k]));
          x[k] = t;
        }
      }
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        unpair2(x[k], f[first(2 * k)], f[first(2 * k + 1)]);
        unpair2(y2[k], f[other(2 * k)], f[other(2 * k + 1)]);
      }
      T* const y = reinterpret_cast<T*>(a.s[kv].y) + n * a.s[kv].yt + h * a.s[kv].yh;
      *reinterpret_cast<uint4*>(y + d0) = pack<T>(f);
      if (second) *reinterpret_cast<uint4*>(y + d1) = pack<T>(f + VEC);
    }
  }
}

// heads, parts, strides or addresses that are no whole vectors: a warp per head, a value at a time
template <typename T, bool PAIRS>
__global__ void __launch_bounds__(THREADS) rotate_any_kernel(const RotArgs a) {
  const int lane = threadIdx.x & 31, total = a.s[0].heads + a.s[1].heads;
  pdl_wait();
  pdl_launch_dependents();
  const long long w = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5), n = w / total;
  if (n >= a.N) return;
  int h = (int)(w % total);
  const int kv = h >= a.s[0].heads, half = a.part / 2;
  h -= kv ? a.s[0].heads : 0;
  const Side& sd = a.s[kv];
  const T* const x = reinterpret_cast<const T*>(sd.x) + n * sd.xt + h * sd.xh;
  const T* const wt = reinterpret_cast<const T*>(sd.w);
  T* const y = reinterpret_cast<T*>(sd.y) + n * sd.yt + h * sd.yh;
  float r = 1.f;
  if (wt) {
    float ss = 0.f;
    for (int d = lane; d < a.D; d += 32) ss = __fmaf_rn(to_f(x[d]), to_f(x[d]), ss);
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
    r = rsqrtf(ss / (float)a.D + a.eps);
  }
  auto value = [&](int d) { return wt ? to_f(x[d]) * r * to_f(wt[d]) : to_f(x[d]); };
  if (half > 0) {
    const long long row = place(a, n) * half;
    for (int j = lane; j < half; j += 32) {
      const int i0 = a.offset + (PAIRS ? 2 * j : j), i1 = PAIRS ? i0 + 1 : i0 + half;
      const float c = __ldg(a.cos_t + row + j), s = a.sign * __ldg(a.sin_t + row + j), u = value(i0), v = value(i1);
      y[i0] = from_f<T>(__fmaf_rn(u, c, -__fmul_rn(v, s)));
      y[i1] = from_f<T>(__fmaf_rn(u, s, __fmul_rn(v, c)));
    }
  }
  for (int j = lane; j < a.D - a.part; j += 32) {
    const int d = j < a.offset ? j : j + a.part;
    y[d] = wt ? from_f<T>(value(d)) : x[d];
  }
}

template <typename T>
int rotate_launch(RotArgs& a, bool pairs, cudaStream_t st_) {
  constexpr int VEC = 16 / sizeof(T);
  const bool norm = a.s[0].w || a.s[1].w;
  const int total = a.s[0].heads + a.s[1].heads;
  bool vec = a.D % VEC == 0 && a.D <= 64 * VEC && a.part % (2 * VEC) == 0 && a.offset % VEC == 0 && st::aligned16(a.cos_t) && st::aligned16(a.sin_t);
  for (const Side& s : a.s)
    if (s.heads) vec = vec && s.xt % VEC == 0 && s.xh % VEC == 0 && s.yt % VEC == 0 && s.yh % VEC == 0 && st::aligned16(s.x) && st::aligned16(s.y) && st::aligned16(s.w);
  const char* who = "st_rotate launch";
  if (!vec) {
    const long long blocks = (a.N * total + THREADS / 32 - 1) / (THREADS / 32);
    ST_REQUIRE(blocks < (1ll << 31), "st_rotate: too many heads");
    return st::launch(who, pairs ? rotate_any_kernel<T, true> : rotate_any_kernel<T, false>, dim3((unsigned)blocks), dim3(THREADS), 0, st_, a);
  }
  a.lanes = 1;
  while (a.lanes * 2 * VEC < a.D) a.lanes *= 2;
  // a token's heads are dealt to more warps while the GPU's (some 32 an SM fit) are not all at work
  const int passes = (total + 32 / a.lanes - 1) / (32 / a.lanes);
  const long long want = 32ll * st::sm_count() / a.N;
  a.parts = (int)(want < 1 ? 1 : want > passes ? passes : want);
  const long long blocks = (a.N * a.parts + THREADS / 32 - 1) / (THREADS / 32);
  ST_REQUIRE(blocks < (1ll << 31), "st_rotate: too many tokens");
  auto kernel = pairs ? (norm ? rotate_kernel<T, true, true> : rotate_kernel<T, true, false>)
                      : (norm ? rotate_kernel<T, false, true> : rotate_kernel<T, false, false>);
  return st::launch(who, kernel, dim3((unsigned)blocks), dim3(THREADS), 0, st_, a);
}
}  // namespace

extern "C" int st_rotate(const void* q, int64_t q_token, int64_t q_head, int64_t Hq, const void* k, int64_t k_token, int64_t k_head,
                         int64_t Hk, int64_t N, int64_t D, int type, const int64_t* positions, int positions_step, const float* cos_t,
                         const float* sin_t, int64_t span, int64_t part, int64_t offset, int interleaved, int inverse, const void* wq,
                         const void* wk, double eps, void* q_out, int64_t qo_token, int64_t qo_head, void* k_out, int64_t ko_token,
                         int64_t ko_head, void* stream) {
  const char* who = "st_rotate";
  ST_REQUIRE(type >= 0 && type <= 2, "%s: type must be 0 (BF16), 1 (FP16) or 2 (float32)", who);
  ST_REQUIRE(N >= 0 && Hq >= 0 && Hk >= 0 && Hq + Hk < (1 << 20), "%s: sizes", who);
  ST_REQUIRE(D >= 1 && D <= 65536 && part >= 0 && part % 2 == 0 && offset >= 0 && offset + part <= D,
             "%s: the rotated part must be an even number of a head's values", who);
  ST_REQUIRE(part == 0 || span >= 1, "%s: an empty table", who);
  if (N == 0 || Hq + Hk == 0) return 0;
  ST_REQUIRE((Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)) && (part == 0 || (positions && cos_t && sin_t)), "%s: null pointer", who);
  RotArgs a = {};
  a.s[0] = {q, q_out, Hq ? wq : nullptr, q_token, q_head, qo_token, qo_head, (int)Hq};
  a.s[1] = {k, k_out, Hk ? wk : nullptr, k_token, k_head, ko_token, ko_head, (int)Hk};
  a.pos = reinterpret_cast<const long long*>(positions);
  a.pos_step = positions_step ? 1 : 0;
  a.cos_t = cos_t; a.sin_t = sin_t; a.span = span;
  a.N = N; a.D = (int)D; a.part = (int)part; a.offset = (int)offset;
  a.eps = (float)eps; a.sign = inverse ? -1.f : 1.f;
  const cudaStream_t st_ = (cudaStream_t)stream;
  return type == 0 ? rotate_launch<__nv_bfloat16>(a, interleaved != 0, st_) : type == 1 ? rotate_launch<__half>(a, interleaved != 0, st_)
                                                                                        : rotate_launch<float>(a, interleaved != 0, st_);
}
