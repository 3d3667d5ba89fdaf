// The epilogue of a product y = act(x W^T + bias) + residual, applied to fp32 sums before the one rounding to BF16.  Shared by the GEMV
// (st_gemv.cu) and the two tcgen05 kernels (st_gemm.cu, st_gemm_pair.cu), whose plain forms are compiled without it.
//   EPI_SWIGLU: W's rows are gate and up in 16-row tiles in turn; row j of the result is silu(gate_j) * up_j
#pragma once
#include "st_common.cuh"

namespace st {
constexpr int EPI_NONE = 0, EPI_RELU = 1, EPI_SILU = 2, EPI_GELU = 3, EPI_GELU_TANH = 4, EPI_SWIGLU = 5;

struct Epi {
  const uint16_t* bias;                            // BF16 [M] or nullptr
  const uint16_t* res; long long res_stride;       // BF16 [B][M, swiglu: M / 2] or nullptr; may be the output
  int act;
  long long rows;                                  // of the result (its row stride): M, or M / 2
};

// st_gemm.cu, st_gemv.cu: what both entry points check
int epi_args(Epi& e, const char* who, const void* bias, int act, const void* res, int64_t res_stride, int64_t M);

#ifdef __CUDACC__
// Relative errors, beside the rounding to BF16 (half a step: 2^-8).  __expf(x): 2 + 1.18 |x| units of 2^-23, so that SiLU at z is off by
// 2^-21 near 0 and 2^-16 at -80, GELU by tanh by as much of its exponent and that exponent's own roundings; beyond the exponential's range the
// quotients go to 0 or z
__device__ __forceinline__ float epi_silu(float z) { return z / (1.f + __expf(-z)); }
// GELU, z Phi(z).  1 + erf(z / sqrt 2) cancels for negative z (0.5 % of it at -4.5, all at -5.4).  Here the tail Phi(-|z|) is t 2^(p(t) - z^2 / (2 ln 2)),
// t = 1 / (1 + 9 |z| / 32), p a polynomial fitted for the least largest error over |z| <= 14 (2^-18.8 of Phi; with the exponent's roundings
// 2^-16.8 at -13, where the result leaves fp32's normal range).  A call of erfcf instead, sixteen of them inlined, took the whole kernel's
// registers: 16384 x 4096 at 300 rows 58 us instead of 41, without an activation 48 instead of 37
__device__ __forceinline__ float epi_gelu(float z) {
  const float a = fabsf(z), t = __fdividef(1.f, __fmaf_rn(0.28125f, a, 1.f));
  float p = __fmaf_rn(0.34369749f, t, -1.0878390f);
  p = __fmaf_rn(p, t, 0.88564104f);
  p = __fmaf_rn(p, t, -0.10954575f);
  p = __fmaf_rn(p, t, 0.69016314f);
  p = __fmaf_rn(p, t, 1.4333152f);
  p = __fmaf_rn(p, t, -3.1554291f);
  float tail;
  asm("ex2.approx.f32 %0, %1;" : "=f"(tail) : "f"(__fmaf_rn(-0.72134752f * a, a, p)));
  tail *= t;
  return z * (z < 0.f ? tail : 1.f - tail);
}
__device__ __forceinline__ float epi_act(int act, float z) {
  switch (act) {                                   // (the same for the whole launch)
    case EPI_RELU: return z < 0.f ? 0.f : z;
    case EPI_SILU: return epi_silu(z);
    case EPI_GELU: return epi_gelu(z);
    case EPI_GELU_TANH: return z / (1.f + __expf(-1.5957691216057308f * z * __fmaf_rn(0.044715f * z, z, 1.f)));      // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
  }
  return z;
}
// the same of sixteen values, one branch for all
__device__ __forceinline__ void epi_act16(int act, float (&z)[16]) {
  switch (act) {
#define ST_ACT(A) case A: _Pragma("unroll") for (int k = 0; k < 16; ++k) z[k] = epi_act(A, z[k]); break;
    ST_ACT(EPI_RELU) ST_ACT(EPI_SILU) ST_ACT(EPI_GELU) ST_ACT(EPI_GELU_TANH)
#undef ST_ACT
  }
}
__device__ __forceinline__ float epi_value(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ uint16_t epi_round(float v) {
  const __nv_bfloat16 h = __float2bfloat16_rn(v);
  return *reinterpret_cast<const uint16_t*>(&h);
}

// Sixteen token columns of a warp's 32 rows, lane = row, as tensor memory hands them out.  `left` of the columns exist, `valid` of the rows
// (a multiple of 16); y, res: this warp's first result row of the first column, columns `rows` / `res_stride` values apart.  Lanes pair up,
// even ones on column c and odd on c + 1 with two rows each, so that a store writes 4 bytes a lane, 64 a column; under EPI_SWIGLU lane l
// and l + 16 (gate and up of a row) pair up the same way.  The residual's words are fetched by a call of their own, so that they can be
// requested a chunk ahead, and before the first store (they may be the same memory); from L2: the threads here have not waited for the
// kernel before themselves, so that a line of theirs in L1 may be older than its writes.
__device__ __forceinline__ void epi_fetch16(const Epi& e, int left, int valid, const uint16_t* res, uint32_t (&r)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = 0u;
  if (!e.res) return;
  if (e.act == EPI_SWIGLU) {
    const int hi = lane >> 4, row = lane & 15;
    if (valid == 32)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (2 * j + hi < left) r[j] = (uint32_t)__ldcg(res + (size_t)(2 * j + hi) * e.res_stride + row);
  } else {
    const int odd = lane & 1, row = lane & ~1;
    if (row < valid)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (2 * j + odd < left) r[j] = __ldcg(reinterpret_cast<const uint32_t*>(res + (size_t)(2 * j + odd) * e.res_stride + row));
  }
}
__device__ __forceinline__ void epi_store16(const Epi& e, const uint32_t (&v)[16], float bias, int left, int valid, uint16_t* y, const uint32_t (&r)[8]) {
  const int lane = threadIdx.x & 31;
  float z[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) z[k] = __uint_as_float(v[k]) + bias;
  if (e.act == EPI_SWIGLU) {
    const int hi = lane >> 4;
    uint16_t* const p = y + (size_t)hi * e.rows + (lane & 15);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float got = __shfl_xor_sync(FULL, hi ? z[2 * j] : z[2 * j + 1], 16);
      const float x = epi_silu(hi ? got : z[2 * j]) * (hi ? z[2 * j + 1] : got) + __uint_as_float(r[j] << 16);
      if (valid == 32 && 2 * j + hi < left) p[(size_t)(2 * j) * e.rows] = epi_round(x);
    }
    return;
  }
  epi_act16(e.act, z);
  const int odd = lane & 1, row = lane & ~1;
  uint16_t* const p = y + (size_t)odd * e.rows + row;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float got = __shfl_xor_sync(FULL, odd ? z[2 * j] : z[2 * j + 1], 1);
    const float x0 = (odd ? got : z[2 * j]) + __uint_as_float(r[j] << 16), x1 = (odd ? z[2 * j + 1] : got) + __uint_as_float(r[j] & 0xFFFF0000u);
    if (row < valid && 2 * j + odd < left) *reinterpret_cast<uint32_t*>(p + (size_t)(2 * j) * e.rows) = pack_bf16(x0, x1);
  }
}

// Four rows 4 lane .. 4 lane + 3 of a 128-row block in one token column (a warp a column).  bias: of these rows; y, res: the block's first
// result row of the column; valid: rows of the block that exist.  `word`: epi_fetch4's
__device__ __forceinline__ uint2 epi_fetch4(const Epi& e, int valid, const uint16_t* res) {
  const int lane = threadIdx.x & 31;
  if (!res || 4 * lane >= valid) return make_uint2(0u, 0u);
  return __ldcg(reinterpret_cast<const uint2*>(res + (e.act == EPI_SWIGLU ? (lane >> 3) * 16 + (lane & 3) * 4 : 4 * lane)));
}
__device__ __forceinline__ void epi_store4(const Epi& e, float4 z, const float (&bias)[4], int valid, uint16_t* y, uint2 word) {
  const int lane = threadIdx.x & 31;
  z.x += bias[0]; z.y += bias[1]; z.z += bias[2]; z.w += bias[3];
  int at = 4 * lane;
  bool mine = at < valid;
  if (e.act == EPI_SWIGLU) {                       // lane ^ 4 holds the same rows of the other projection
    float4 up;
    up.x = __shfl_xor_sync(FULL, z.x, 4); up.y = __shfl_xor_sync(FULL, z.y, 4); up.z = __shfl_xor_sync(FULL, z.z, 4); up.w = __shfl_xor_sync(FULL, z.w, 4);
    z.x = epi_silu(z.x) * up.x; z.y = epi_silu(z.y) * up.y; z.z = epi_silu(z.z) * up.z; z.w = epi_silu(z.w) * up.w;
    mine = mine && !(lane & 4);
    at = (lane >> 3) * 16 + (lane & 3) * 4;
  } else {
    z.x = epi_act(e.act, z.x); z.y = epi_act(e.act, z.y); z.z = epi_act(e.act, z.z); z.w = epi_act(e.act, z.w);
  }
  if (!mine) return;
  *reinterpret_cast<uint2*>(y + at) = make_uint2(pack_bf16(z.x + __uint_as_float(word.x << 16), z.y + __uint_as_float(word.x & 0xFFFF0000u)),
                                                 pack_bf16(z.z + __uint_as_float(word.y << 16), z.w + __uint_as_float(word.y & 0xFFFF0000u)));
}
__device__ __forceinline__ void epi_bias4(const Epi& e, long long row0, int valid, float (&bias)[4]) {
  const int lane = threadIdx.x & 31;
  const bool has = e.bias && 4 * lane < valid;
#pragma unroll
  for (int k = 0; k < 4; ++k) bias[k] = has ? epi_value(__ldg(e.bias + row0 + 4 * lane + k)) : 0.f;
}
#endif
}  // namespace st
