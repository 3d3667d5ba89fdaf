// The 8-bit KV page shared by its kernels (st_kv8.cu, st_kv8_chunk.cu).
//
// Page: uint8 [blocks, H, 2 (K/V), 16, D] e4m3 codes and int8 exps [blocks, H, 2]; value = e4m3(code) * 2^exp, exp in [E8_MIN, E8_MAX].
// A power of two, because the codes are floating point: a finer scale would not make them more precise, and a page whose largest value
// grows as tokens arrive changes its exponent without rounding again (but for codes that become subnormal).  Every value has four
// significant bits, so it is a BF16 number (and the code an FP16 one) exactly and the tensor cores read it without a rounding.
//
// At D = 128 the 16-byte pieces of a row are kept in another order (piece8): rows are 128 B apart, and both ways in which a warp of the
// decode kernel reads a page (eight rows x four pieces for keys, four even or odd rows x two pieces for values) then touch every bank
// of shared memory once per eight lanes.
#pragma once
#include "st_common.cuh"

namespace st {
constexpr int E8_MIN = -64, E8_MAX = 56;

template <int D>
__device__ __forceinline__ int piece8(int row, int c) {
  return D == 128 ? c ^ (row & 6) ^ ((row & 1) << 2) : c;
}
template <int D>
__device__ __forceinline__ size_t page8_off(long long blk, int H, int h, int kvi) {
  return (((size_t)blk * H + h) * 2 + kvi) * (PAGE * D);
}
__device__ __forceinline__ int page8_exp(int e) { return min(max(e, E8_MIN), E8_MAX); }
// 2^e, e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// Four codes -> their BF16 bit patterns times 2^-120: the four exponent and three mantissa bits are put at the low end of BF16's
// exponent field and the top of its mantissa, subnormal codes becoming subnormals, so the value is exact without a multiplication;
// 2^120 goes into a factor that is applied anyway.  High bytes hi = s0000eee, low bytes lo = emmm0000.
// (The codes 0x7F and 0xFF, not a number in e4m3, are written by no append; here they read as +-480.)
__device__ __forceinline__ void codes_split(uint32_t w, uint32_t& lo, uint32_t& hi) {
  hi = ((w & 0x70707070u) >> 4) | (w & 0x80808080u);
  lo = (w & 0x0F0F0F0Fu) << 4;
}
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t& p01, uint32_t& p23) {
  uint32_t lo, hi;
  codes_split(w, lo, hi);
  p01 = __byte_perm(lo, hi, 0x5140);
  p23 = __byte_perm(lo, hi, 0x7362);
}
// the value of a BF16 pattern from codes_to_bf16 (low or high half) without its 2^-120 and with 2^e
__device__ __forceinline__ float2 codes_value(uint32_t p, float up) {      // up = 2^(20 + e)
  constexpr float C = 1.2676506002282294e30f;                             // 2^100
  return make_float2(__uint_as_float(p << 16) * C * up, __uint_as_float(p & 0xFFFF0000u) * C * up);
}
// two codes -> FP16, exact: the low and the high half of a word
__device__ __forceinline__ uint32_t f16_low(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t f16_high(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 2^x, relative error below 2^-22, results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// q * 2^-e has its largest magnitude (fp32 bits `most`) in [2^13, 2^14); 0 for zeros; at least -100, so that 2^-e is a number
__device__ __forceinline__ int q_exp(uint32_t most) {
  return most < 0x00800000u ? 0 : max(min((int)(most >> 23) - 127, 126) - 13, -100);
}

// the reference that probabilities are relative to (base 2, P = 2^(x - r)): between UNDER8 and RAISE8 below the largest x
constexpr float UNDER8 = 7.f, RAISE8 = 15.f;

// ---- the attention's arguments
struct Attn8 {
  const uint16_t* q; long long q_stride;
  const int* cu;                                   // first query of each sequence [B + 1]; nullptr: one query each
  const uint8_t* kv; const int8_t* exps; long long nblocks;
  const int* table; long long table_stride;        // rows of table_width entries
  const int* lens; const int* starts;
  uint16_t* out; long long out_stride;
  float scale_log2;
  int B, Hq, H, window, table_width;
  long long T;
};
// partial results of sequences that are split: o [T, Hq, splits, D] (not normalised), ml [T, Hq, splits, 2] = (reference, base 2; sum)
// (decode kernel: o = nullptr, the splits of a unit are a cluster that joins on chip)
struct Parts8 { float* o; float* ml; int splits, min_pages; };

// A CTA's rows, the same in all of its threads: rows row0 .. row0 + rows - 1 of the n * G rows (query, head of the group) of sequence b,
// whose first query is row `first` of q
// (and its length and first valid token, requested beside the row counts)
struct Rows8 { int b, row0, rows, first, n, len, start; };
// tile `slot` of TILE rows, sequences' tiles one after the other; false: there is none
template <int TILE>
__device__ __forceinline__ bool find_rows(const Attn8& a, int G, int slot, int lane, Rows8& w) {
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    int lo = 0, n = 0, len = 0, start = 0;
    if (b < a.B) {
      len = a.lens[b];
      start = a.starts ? max(a.starts[b], 0) : 0;
      lo = a.cu ? a.cu[b] : b;
      n = a.cu ? a.cu[b + 1] - lo : 1;
      if (lo < 0 || n < 0 || lo + (long long)n > a.T) n = 0;      // (not inside q: no work)
    }
    const int mine = (int)(((long long)n * G + TILE - 1) / TILE);
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(FULL, sum, o);
      if (lane >= o) sum += v;
    }
    const int begin = before + sum - mine;
    const unsigned hit = __ballot_sync(FULL, slot >= begin && slot < begin + mine);
    if (hit) {
      const int src = __ffs(hit) - 1;
      w.b = b0 + src;
      w.first = __shfl_sync(FULL, lo, src);
      w.n = __shfl_sync(FULL, n, src);
      w.len = __shfl_sync(FULL, len, src);
      w.start = __shfl_sync(FULL, start, src);
      w.row0 = (slot - __shfl_sync(FULL, begin, src)) * TILE;
      w.rows = min(TILE, w.n * G - w.row0);
      return true;
    }
    before += __shfl_sync(FULL, sum, 31);
  }
  return false;
}

// st_kv8.cu: what both forms of the attention check and pass on; the join of the partial results
int attn8_args(Attn8& a, const char* who, const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv,
               const int8_t* exps, int64_t nblocks, int64_t Hkv, int64_t D, const int32_t* bt, int64_t btw, int64_t bts, const int32_t* lens,
               const int32_t* starts, int64_t window, void* out, int64_t os, double scale);
// Chunks of few rows per sequence go through the decode kernel, eight rows a CTA: its time grows with every eight rows, the chunk kernel's
// hardly up to 128.  32 sequences of 2000 tokens, D = 128, us: 16 rows 38 in the decode kernel and 103 in the other, 32 rows 63 and 74, 64
// rows 119 and 75.  D = 64: 28 rows 15 and 30, 56 rows 27 and 30, 112 rows 46 and 31.  By the mean over the sequences, which is what the host
// knows: a batch of decode tokens with one long chunk is faster as two calls.  (chunk_splits8 in kvcache.py states the same bound.)
constexpr int FEW_ROWS = 32;
inline bool few_rows8(long long T, long long B, long long G) { return T * G <= FEW_ROWS * B; }
int rows8_attn(const char* who, const Attn8& a, const Parts8& parts, int D, cudaStream_t stream);
int merge8(const char* who, const Attn8& a, const Parts8& parts, int D, cudaStream_t stream);
}  // namespace st
