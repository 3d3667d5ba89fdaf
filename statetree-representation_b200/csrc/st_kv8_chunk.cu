// Causal attention of several query tokens per sequence over 8-bit KV pages, on the tensor cores (tcgen05).
//
// A row is a (query token, head) pair of one KV head's group, so a CTA's 256 rows (two accumulator tiles of 128) are 256 / G
// consecutive tokens of one sequence, whatever G is; keys come 128 at a time (eight pages):
//     S = Q K^T   128 x 128, A and B from shared memory            P = exp2(S * c - m) in FP16, back into S's tensor-memory columns
//     O += P V    128 x D, A = P from tensor memory, B = V from shared memory as it lies (dims contiguous: MN-major)
// Warps: eight of softmax (a thread owns one row, so its maximum and sum need no other thread), four that bring pages into shared memory
// by bulk copies and turn their codes into FP16 operand tiles, one that issues the MMAs.  While one tile's softmax
// runs, the tensor core works on the other's: S0 P0 S1 P1 ... in turn.
// Tensor memory: S0, S1 (128 columns each; P takes the first 64 of its own), O0, O1 (D each).
//
// Types and scales as in the decode kernel: e4m3 codes are FP16 numbers (one instruction converts two; as BF16 patterns the integer
// operations of the converters were the limit beside the softmax), a row of q is scaled by a power of two so that FP16 holds its eight
// bits, a page's key exponent is a factor of its sixteen score columns, its value exponent joins the softmax exponent of its sixteen
// columns of P and is taken out of the sum per page.  P is rounded to FP16 (2^-11 of each at most, and 2^-32 of the largest), everything
// else but the output is fp32.
//
// Measured (32 query heads, 8 KV heads, D = 128): 2048 queries behind 30000 tokens 1.00-1.05 ms = 1.0 PFLOP/s, a prompt of 4096 tokens 172 us.
// A key tile takes 2.3 us for the 256 rows: a row tile's softmax about 2300 cycles, its MMAs and the hand-overs 1200, of which the other
// row tile's overlap most; the MMAs by themselves 2270 cycles for both.  Shared memory is busy 2560 of its cycles (operands 192 KB,
// conversion 128 KB).  A CTA costs about 8 us besides (look-ups, q, first pages, output).
#include <float.h>
#include <math.h>

#include <atomic>

#include "../../include/statetree_b200.h"
#include "st_host.h"
#include "st_kv8.cuh"
#include "st_tc.cuh"

namespace {
using namespace st;

constexpr int KEYS = 128, TILE_PAGES = KEYS / PAGE, ROWS = 128;
constexpr int W_CONV = 8, W_MMA = 12, WARPS = 16;                 // softmax warps 0 .. 7 (tile = warp / 4); 13 .. 15 only lend registers
constexpr int CRING = 4;                                          // page factors of so many key tiles are kept

template <int D>
struct Lay {                                                      // shared memory
  static constexpr int HALF = 128 * 128;                          // 128 rows x 64 FP16, 128-byte swizzle
  static constexpr int TILE = D / 64 * HALF;
  static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE;         // two tiles of Q, two stages of K and V
  static constexpr int RAW = 6 * TILE, UNIT = PAGE * D;           // codes of one key tile: its keys, its values
  static constexpr int F = RAW + 2 * TILE_PAGES * UNIT, BARS = F + CRING * TILE_PAGES * 3 * 4;
  static constexpr int NBARS = 25, SLOT = BARS + NBARS * 8;
  // (more than half of an SM's shared memory: one CTA per SM, which holds all of its tensor memory)
  static constexpr int BYTES = (SLOT + 16 > 120 * 1024 ? SLOT + 16 : 120 * 1024) + 1024;
};

struct Chunk8 { Attn8 a; Parts8 parts; int* status; int slots; };

// Shared-memory operands.  Descriptor: address / 16 and the stride of the leading dimension / 16 in the low word; in the high one the
// stride of 8-row groups (1024 B), the version and the 128-byte swizzle, the same for all of them.  So the issuing thread keeps the low
// words and adds to them (with whole descriptors formed at every MMA the issue took as long as the MMAs).
//   K-major (Q, K: a row holds 64 values of the contracted dimension)   leading stride unused
//   MN-major (V: a row, one key, holds 64 values of the other one)       the next 64 values `next` bytes further
constexpr uint32_t DESC_HI = 64u | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_k(uint32_t saddr) { return (saddr & 0x3FFFFu) >> 4 | 1u << 16; }
__device__ __forceinline__ uint32_t desc_mn(uint32_t saddr, uint32_t next) { return (saddr & 0x3FFFFu) >> 4 | (next >> 4) << 16; }
// D (+)= A B^T, A from shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}"
               :: "r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(DESC_HI) : "memory");
}
// the same, A from tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}"
               :: "r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(DESC_HI) : "memory");
}
#define ST_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define ST_I4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t* v) {            // (complete after tm_wait_ld)
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
               "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : ST_R4(v, 0), ST_R4(v, 4), ST_R4(v, 8), ST_R4(v, 12), ST_R4(v, 16), ST_R4(v, 20), ST_R4(v, 24), ST_R4(v, 28)
               : "r"(addr));
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : ST_R4(v, 0), ST_R4(v, 4), ST_R4(v, 8), ST_R4(v, 12) : "r"(addr));
}
template <int N>
__device__ __forceinline__ void tm_wait_ld(uint32_t* v) {                        // (v's readers stay behind the wait)
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int k = 0; k < N; ++k) asm volatile("" : "+r"(v[k]));
}
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pair2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2f(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               :: "r"(addr), ST_I4(v, 0), ST_I4(v, 4), ST_I4(v, 8), ST_I4(v, 12) : "memory");
}
#undef ST_R4
#undef ST_I4
// registers of a warpgroup: 512 threads start with 128 each (64 K in all, the SM's); 2 x 184 + 96 + 48 = 4 x 128
constexpr int R_SOFTMAX = 184, R_CONV = 96, R_MMA = 48;
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }

// What a CTA works on; the same in all of its threads
struct Work : Rows8 {
  int h, split, pos0;                                             // position of query 0
  int lo0, first_tile, tiles, count0, count1;                           // key tiles of the split; of those, how many each row tile needs
};

template <int D>
__global__ void __launch_bounds__(WARPS * 32, 1) kv8_chunk_kernel(const Chunk8 c) {
  using L = Lay<D>;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t *const begin1 = bars, *const kfull = bars + 2, *const vfull = bars + 4, *const sfull = bars + 6, *const pfull = bars + 8,
           *const ofull = bars + 12, *const empty = bars + 14, *const raw = bars + 16;           // pfull: [half of the keys][row tile]
  uint64_t* const drain = bars + 24;                              // raw: [converter warp][keys, values]
  uint32_t* const slot_at = reinterpret_cast<uint32_t*>(smem + L::SLOT);
  const Attn8& a = c.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.Hq / a.H;
  pdl_wait();
  pdl_launch_dependents();

  // ---- what this CTA works on.  Later tiles of a sequence see more keys: they go first
  Work w;
  {
    int x = blockIdx.x;
    w.split = x % c.parts.splits;
    x /= c.parts.splits;
    w.h = x % a.H;
    if (!find_rows<2 * ROWS>(a, G, c.slots - 1 - x / a.H, lane, w)) return;
    const int start = w.start;
    w.pos0 = w.len - w.n;
    const int first_pos = w.pos0 + w.row0 / G, last_pos = w.pos0 + (w.row0 + w.rows - 1) / G;
    w.lo0 = start;
    const int lo = a.window > 0 ? max(start, first_pos - a.window + 1) : start;
    const int end = (int)min((long long)last_pos + 1, (long long)a.table_width * PAGE);            // keys [lo, end)
    const int t0 = lo / KEYS, t1 = end > lo ? (end - 1) / KEYS + 1 : t0;
    const int per = (t1 - t0 + c.parts.splits - 1) / c.parts.splits;
    w.first_tile = t0 + w.split * per;
    w.tiles = max(0, min(t1, w.first_tile + per) - w.first_tile);
    const int mid_pos = w.pos0 + (w.row0 + min(w.rows, ROWS) - 1) / G;                   // last position of the first row tile
    w.count0 = mid_pos < 0 ? 0 : max(0, min(w.tiles, mid_pos / KEYS + 1 - w.first_tile));
    w.count1 = w.rows > ROWS ? w.tiles : 0;
  }
  const int tiles = max(w.count0, w.count1);
  // (pages behind the last key of the sequence, or behind its row of the table, may not exist: no key of theirs is seen)
  const int end_page = min((w.pos0 + w.n - 1) / PAGE + 1, a.table_width);
  const uint64_t keep = policy_evict_last();                      // other row tiles of the sequence read the same pages

  if (warp == W_MMA) {
    if (elect_one()) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(kfull + i, 4);
        mbar_init(vfull + i, 4);
        mbar_init(sfull + i, 1);
        mbar_init(pfull + i, 4);
        mbar_init(pfull + 2 + i, 4);
        mbar_init(ofull + i, 1);
        mbar_init(empty + i, 1);
      }
      mbar_init(drain, 1);
      mbar_init(begin1, 4);
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc<1>(slot_at, 512);
    tmem_relinquish<1>();
  }
  // (each role has something to request before it needs the others: the rows of q, the first pages)
  auto meet = [] {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };

  if (warp < W_CONV) {
    regs_up<R_SOFTMAX>();
    // ---------------------------------------------------------------- softmax: this thread's row
    const int t = warp >> 2, my = w.row0 + t * ROWS + (warp & 3) * 32 + lane, count = t ? w.count1 : w.count0;
    const bool live = my < w.row0 + w.rows;
    const int token = live ? my / G : 0, head = live ? my % G : 0, hq = w.h * G + head;
    const int pos = w.pos0 + token;
    // (a row that is none sees everything: its results go nowhere, and a warp with one does not take the masked way for it)
    const int hi = live ? min(pos, a.table_width * PAGE - 1) : 0x7FFFFFFF, lo = !live ? 0 : a.window > 0 ? max(w.lo0, pos - a.window + 1) : w.lo0;
    const bool any = __any_sync(FULL, live);
    float m = -INFINITY, l = 0.f, q_up = 1.f;                     // q_up undoes the scale of q
    bool ok = true;
    // ---- the warp's 32 rows of q as FP16, each times a power of two that its largest value asks for: D / 8 lanes read a row
    if (count > 0) {
      constexpr int LANES = D / 8, PER = 32 / LANES;
      const long long mine = live ? (long long)(w.first + token) * a.q_stride + (long long)hq * D : -1;
      const int c = lane % LANES;
      uint8_t* const rows = smem + L::Q + t * L::TILE + (warp & 3) * (32 * 128) + (c >> 3) * L::HALF;
      uint4 u[LANES];
#pragma unroll
      for (int i = 0; i < LANES; ++i) {
        const long long from = __shfl_sync(FULL, mine, i * PER + lane / LANES);
        u[i] = from >= 0 ? *reinterpret_cast<const uint4*>(a.q + from + 8 * c) : make_uint4(0, 0, 0, 0);
      }
      int e_mine = 0;
#pragma unroll
      for (int i = 0; i < LANES; ++i) {
        uint32_t x[4] = {u[i].x, u[i].y, u[i].z, u[i].w}, most = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max(most, max(x[k] << 16 & 0x7FFF0000u, x[k] & 0x7FFF0000u));
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(FULL, most, o));
        const int e = q_exp(most), theirs = __shfl_sync(FULL, e, (lane % PER) * LANES);
        if (lane / PER == i) e_mine = theirs;
        const float down = pow2i(-e);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = pack_f16(__uint_as_float(x[k] << 16) * down, __uint_as_float(x[k] & 0xFFFF0000u) * down);
        const int r = i * PER + lane / LANES;
        *reinterpret_cast<uint4*>(rows + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
      }
      q_up = pow2i(e_mine);
      fence_proxy_async();
    }
    meet();
    const uint32_t tmem = *slot_at + ((uint32_t)((warp & 3) * 32) << 16), ts = tmem + t * 128, to = tmem + 256 + t * D;
    // The second row tile begins when the first has its first P: from then on each has the special function units to itself while the
    // other's products run.  (A barrier of its own, which completes once: the first tile's softmax does not wait for this one's, so that
    // it could complete a phase of `pfull` and the next before a warp here has looked)
    if (t == 1 && count > 0 && w.count0 > 0) ok = mbar_wait(begin1, 0);
    for (int j = 0; ok && j < count; ++j) {
      if (!mbar_wait_look(sfull + t, (uint32_t)j & 1u)) { ok = false; break; }
      tc_fence_after();
      if (any) {
        const float* const fac = reinterpret_cast<const float*>(smem + L::F) + (j % CRING) * (TILE_PAGES * 3);
        const int k0 = (w.first_tile + j) * KEYS, l0 = lo - k0, l1 = hi - k0;                // this row sees columns l0 .. l1
        // ---- the row's scores, all 128 in registers; what it does not see is -inf
        uint32_t v[KEYS];
#pragma unroll
        for (int q = 0; q < 4; ++q) tm_ld32(ts + 32 * q, v + 32 * q);
        tm_wait_ld<KEYS>(v);
        if (__any_sync(FULL, l0 > 0 || l1 < KEYS - 1)) {
#pragma unroll
          for (int k = 0; k < KEYS; ++k) v[k] = k < l0 || k > l1 ? 0xFF800000u : v[k];
        }
        float top = -INFINITY, by[TILE_PAGES];
#pragma unroll
        for (int p = 0; p < TILE_PAGES; ++p) {
          by[p] = fminf(fmaf(fac[p], q_up, FLT_MIN), 3e38f);       // (not 0: it multiplies the -inf of what the row does not see)
          float x = max3(__uint_as_float(v[16 * p]), __uint_as_float(v[16 * p + 1]), __uint_as_float(v[16 * p + 2]));
          float y = max3(__uint_as_float(v[16 * p + 3]), __uint_as_float(v[16 * p + 4]), __uint_as_float(v[16 * p + 5]));
#pragma unroll
          for (int k = 6; k < 14; k += 4) {
            x = max3(x, __uint_as_float(v[16 * p + k]), __uint_as_float(v[16 * p + k + 1]));
            y = max3(y, __uint_as_float(v[16 * p + k + 2]), __uint_as_float(v[16 * p + k + 3]));
          }
          x = max3(x, __uint_as_float(v[16 * p + 14]), __uint_as_float(v[16 * p + 15]));
          top = fmaxf(top, fmaf(fmaxf(x, y), by[p], fac[TILE_PAGES + p]));
        }
        if (__any_sync(FULL, top > m + RAISE8)) {
          const float up = fmaxf(m, top - UNDER8), f = up == m ? 1.f : ex2(m - up);
          m = up;
          l *= f;
          if (j > 0) {                                            // (O's product of the tile before has completed: sfull says so)
#pragma unroll
            for (int q = 0; q < D / 16; ++q) {
              uint32_t o[16];
              tm_ld16(to + 16 * q, o);
              tm_wait_ld<16>(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tm_st16(to + 16 * q, o);
            }
          }
        }
        // ---- P, and the sum
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int pg = 2 * q + p;
            const float add = fac[TILE_PAGES + pg] - ref;
            const uint64_t by2 = pair2(by[pg], by[pg]), add2 = pair2(add, add);
            uint64_t sum = 0;
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              float x0, x1;
              unpair2(fma2(pair2(__uint_as_float(v[16 * pg + k]), __uint_as_float(v[16 * pg + k + 1])), by2, add2), x0, x1);
              x0 = ex2(x0);
              x1 = ex2(x1);
              sum = add2f(sum, pair2(x0, x1));
              pk[8 * p + k / 2] = pack_f16(x0, x1);
            }
            float s0, s1;
            unpair2(sum, s0, s1);
            l = fmaf(s0 + s1, fac[2 * TILE_PAGES + pg], l);
          }
          tm_st16(ts + 16 * q, pk);
          if (q == 1) {                                           // the product with the first 64 keys need not wait for the others
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull + t);
          }
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (!any) mbar_arrive(pfull + t);
        mbar_arrive(pfull + 2 + t);
        if (t == 0 && j == 0) mbar_arrive(begin1);
      }
    }
    if (ok && count > 0) ok = mbar_wait(ofull + t, 0);
    if (!ok && lane == 0) atomicExch(c.status, ERR_WAIT_ACC);
    // ---- out.  (a wait that ran out leaves the rows unwritten)
    if (ok && any) {
      tc_fence_after();
      const long long r = (long long)(w.first + token) * a.Hq + hq;
      const float inv = c.parts.splits > 1 ? 1.f : (l > 0.f ? 1.f / l : l);
      if (live && c.parts.splits > 1) {
        float* const ml = c.parts.ml + (r * c.parts.splits + w.split) * 2;
        ml[0] = l > 0.f || l != l ? m : -INFINITY;
        ml[1] = l;
      }
      if (c.parts.splits > 1) {
        float* const o = c.parts.o + (r * c.parts.splits + w.split) * D;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t v[32];
          if (count > 0) {
            tm_ld32(to + 32 * q, v);
            tm_wait_ld<32>(v);
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = count > 0 && l != 0.f ? __float_as_uint(__uint_as_float(v[k]) * inv) : 0u;
          if (live)
#pragma unroll
            for (int k = 0; k < 8; ++k) reinterpret_cast<uint4*>(o + 32 * q)[k] = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          __syncwarp();
        }
      } else {
        // the warp's rows leave through where its rows of q were (their last scores are done), D / 8 lanes a row
        constexpr int LANES = D / 8, PER = 32 / LANES;
        uint8_t* const rows = smem + L::Q + t * L::TILE + (warp & 3) * (32 * 2 * D);
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t v[32];
          if (count > 0) {
            tm_ld32(to + 32 * q, v);
            tm_wait_ld<32>(v);
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = count > 0 && l != 0.f ? __float_as_uint(__uint_as_float(v[k]) * inv) : 0u;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = pack_bf16(__uint_as_float(v[8 * k + 2 * i]), __uint_as_float(v[8 * k + 2 * i + 1]));
            *reinterpret_cast<uint4*>(rows + lane * (2 * D) + (((4 * q + k) ^ (lane & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
        __syncwarp();
        const long long mine = live ? (long long)(w.first + token) * a.out_stride + (long long)hq * D : -1;
#pragma unroll
        for (int i = 0; i < LANES; ++i) {
          const int row = i * PER + lane / LANES;
          const long long out = __shfl_sync(FULL, mine, row);
          if (out >= 0)
            *reinterpret_cast<uint4*>(a.out + out + 8 * (lane % LANES)) =
                *reinterpret_cast<const uint4*>(rows + row * (2 * D) + (((lane % LANES) ^ (row & 7)) << 4));
        }
      }
    }
    tc_fence_before();
  } else if (warp < W_MMA) {
    regs_down<R_CONV>();
    // ---------------------------------------------------------------- converters: codes -> operand tiles.  A warp brings in and
    // converts pages cw and cw + 4 of every key tile by itself: a bulk copy per page of keys or values, the next one under way as soon as
    // this one is in registers.  (Plain loads in flight would be waited for by the proxy fence behind every tile: 1000 cycles each.)  A
    // lane's 16-byte piece becomes two of a tile row; eight lanes read four pieces of an even row and four of the next, and store them
    // so, which with the page's order of pieces and the tiles' swizzle meets every bank once.
    constexpr int STEP = 512 / D, STEPS = PAGE / STEP;            // rows of a page that a warp takes at once
    const int cw = warp - W_CONV;
    const int r = D == 128 ? 2 * (lane >> 4) + ((lane >> 2) & 1) : lane >> 2;
    const int lc = D == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;
    uint8_t* const mine = smem + L::RAW + cw * (4 * L::UNIT);     // [keys, values][page cw, page cw + 4]
    uint64_t* const my_raw = raw + 2 * cw;
    const uint8_t* const head_pages = a.kv + page8_off<D>(0, a.H, w.h, 0);
    const size_t page_step = (size_t)a.H * (2 * L::UNIT);
    const int* const table = a.table + (long long)w.b * a.table_stride;
    // lane l holds entry and exponents of page cw + 4 (l % 2) of the sixteen key tiles' (l / 2)-th; the next sixteen are requested
    // half way; -1 = there is no such page
    auto entry = [&](int j) {
      const int t = j + (lane >> 1), p = (w.first_tile + t) * TILE_PAGES + cw + 4 * (lane & 1);
      if (t >= tiles || p >= end_page) return -1;
      const int e = __ldg(table + p);
      return e < 0 ? 0 : (int)min((long long)e, a.nblocks - 1);
    };
    auto exps_of = [&](int e) -> uint32_t {
      return e >= 0 ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(a.exps) + (size_t)e * a.H + w.h) : 0u;
    };
    if (lane == 0) {
      mbar_init(my_raw, 1);
      mbar_init(my_raw + 1, 1);
      fence_barrier_init();
    }
    __syncwarp();
    int now = entry(0), next = -1;
    uint32_t now_x = exps_of(now), next_x = 0;
    auto fetch = [&](int j, int kvi, int e) {                     // e: the entries of tile j's sixteen
      const int e0 = __shfl_sync(FULL, e, 2 * (j & 15)), e1 = __shfl_sync(FULL, e, 2 * (j & 15) + 1);
      uint8_t* const to = mine + kvi * (2 * L::UNIT);
      if (elect_one()) {
        mbar_expect_tx(my_raw + kvi, (uint32_t)(((e0 >= 0) + (e1 >= 0)) * L::UNIT));
        if (e0 >= 0) bulk_g2s(to, head_pages + e0 * page_step + kvi * L::UNIT, L::UNIT, my_raw + kvi, keep);
        if (e1 >= 0) bulk_g2s(to + L::UNIT, head_pages + e1 * page_step + kvi * L::UNIT, L::UNIT, my_raw + kvi, keep);
      }
      __syncwarp();
    };
    if (tiles > 0) {
      fetch(0, 0, now);
      fetch(0, 1, now);
    }
    meet();
    bool ok = true;
    for (int j = 0; ok && j < tiles; ++j) {
      const int s = j & 1, at = 2 * (j & 15);
      if ((j & 15) == 4) next = entry((j & ~15) + 16);
      if ((j & 15) == 12) next_x = exps_of(next);
      const int ahead = (j & 15) == 15 ? next : now;
      const int have[2] = {__shfl_sync(FULL, now, at), __shfl_sync(FULL, now, at + 1)};
      const uint32_t x0 = __shfl_sync(FULL, now_x, at), x1 = __shfl_sync(FULL, now_x, at + 1);
      if (lane < 2) {                                             // factors of the two pages
        float* const fac = reinterpret_cast<float*>(smem + L::F) + (j % CRING) * (TILE_PAGES * 3) + cw + 4 * lane;
        const uint32_t x = lane ? x1 : x0;
        const int ek = page8_exp((int8_t)(x & 0xFF)), ev = page8_exp((int8_t)(x >> 8));
        fac[0] = a.scale_log2 * pow2i(ek);
        fac[TILE_PAGES] = (float)ev;
        fac[2 * TILE_PAGES] = pow2i(-ev);
      }
      __syncwarp();
#pragma unroll
      for (int kvi = 0; kvi < 2; ++kvi) {
        if (ok) ok = mbar_wait_look(my_raw + kvi, (uint32_t)j & 1u);
        if (!ok) break;
        uint4 buf[2][STEPS];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            const int row = STEP * i + r;
            buf[p][i] = make_uint4(0, 0, 0, 0);                   // (a page that is not there: zeros)
            if (have[p] >= 0) buf[p][i] = *reinterpret_cast<const uint4*>(mine + (2 * kvi + p) * L::UNIT + row * D + 16 * piece8<D>(row, lc));
          }
        __syncwarp();
        if (j + 1 < tiles) {
          fence_proxy_async();
          fetch(j + 1, kvi, ahead);
        }
        // K's stage is free when the scores of tile j - 2 are, V's when its products are: see the commits of the MMA loop
        const int e = kvi ? j - 1 : j - 2;
        if (j > 1) ok = mbar_wait_look(empty + (e & 1), (uint32_t)(e >> 1) & 1u);
        if (!ok) break;
        uint8_t* const tile = smem + (kvi ? L::V : L::K) + s * L::TILE + (lc >> 2) * L::HALF;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            const uint4 u = buf[p][i];
            const uint32_t o[8] = {f16_low(u.x), f16_high(u.x), f16_low(u.y), f16_high(u.y),
                                   f16_low(u.z), f16_high(u.z), f16_low(u.w), f16_high(u.w)};
            const int row = (cw + 4 * p) * PAGE + STEP * i + r;
            const uint32_t u0 = (uint32_t)((((lc & 3) * 2) ^ (row & 7)) << 4);
            uint8_t* const to = tile + row * 128;
            *reinterpret_cast<uint4*>(to + u0) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(to + (u0 ^ 16)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive((kvi ? vfull : kfull) + s);
      }
      if ((j & 15) == 15) {
        now = next;
        now_x = next_x;
      }
    }
    if (!ok) {
      if (lane == 0) atomicExch(c.status, ERR_WAIT_EMPTY);
      for (int i = 0; i < 4; ++i) (void)mbar_wait(my_raw + (i >> 1), (uint32_t)i & 1u);      // (copies in flight land before the CTA ends)
    }
  } else {
    regs_down<R_MMA>();
    if (warp == W_MMA) {
    // ---------------------------------------------------------------- MMAs.  One thread's MMAs complete in the order of their issue
    // (and a commit covers all before it): S of the next key tile may take the place of the P that the product before it reads
    // (mma_idesc's operands are BF16; FP16 is type 0)
    constexpr uint32_t FP16 = ~(1u << 7 | 1u << 10), IDESC_S = mma_idesc(128, KEYS) & FP16, IDESC_O = (mma_idesc(128, D) & FP16) | 1u << 16;
    meet();
    const uint32_t tmem = *slot_at;
    // The whole loop runs in one elected thread, waits included: a warp that meets again around each step costs more than the steps
    if (elect_one()) {
      const uint32_t dq = desc_k(smem_addr(smem + L::Q)), dk = desc_k(smem_addr(smem + L::K)), dv = desc_mn(smem_addr(smem + L::V), L::HALF);
      auto scores = [&](int t, int s) {
        const uint32_t q = dq + t * (L::TILE >> 4), k = dk + s * (L::TILE >> 4);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t at = (i >> 2) * (L::HALF >> 4) + 2 * (i & 3);
          mma_ss(tmem + t * 128, q + at, k + at, IDESC_S, i > 0);
        }
        tc_commit(sfull + t);
      };
      auto outputs = [&](int t, int s, int half, bool more) {
        const uint32_t v = dv + s * (L::TILE >> 4);
#pragma unroll
        for (int k = 0; k < KEYS / 32; ++k) {
          const int i = half * (KEYS / 32) + k;
          mma_ts(tmem + 256 + t * D, tmem + t * 128 + 8 * i, v + i * (2048 >> 4), IDESC_O, more || i > 0);
        }
      };
      // Three commits a key tile (each waits for the one before it): the scores of either row tile, and `empty`, behind the first
      // product of tile j, which says that the scores of tile j and the products of tile j - 1 are done: K(j) and V(j - 1) are free
      bool ok = true;
      if (tiles > 0) {
        ok = mbar_wait(kfull, 0);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && (t ? w.count1 : w.count0) > 0) {
            tc_fence_after();
            scores(t, 0);
          }
      }
      for (int j = 0; ok && j < tiles; ++j) {
        const int s = j & 1, s1 = s ^ 1;
        ok = mbar_wait_look(vfull + s, (uint32_t)(j >> 1) & 1u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int count = t ? w.count1 : w.count0;
          if (!ok || j >= count) continue;
          ok = mbar_wait_look(pfull + t, (uint32_t)j & 1u);
          if (!ok) continue;
          tc_fence_after();
          outputs(t, s, 0, j > 0);
          ok = mbar_wait_look(pfull + 2 + t, (uint32_t)j & 1u);
          if (!ok) continue;
          tc_fence_after();
          outputs(t, s, 1, true);
          if (t == 0 || j >= w.count0) tc_commit(empty + s);
          if (j + 1 < count) {
            ok = mbar_wait_look(kfull + s1, (uint32_t)((j + 1) >> 1) & 1u);
            if (!ok) continue;
            tc_fence_after();
            scores(t, s1);
          } else {
            tc_commit(ofull + t);
          }
        }
      }
      if (!ok) {                                                  // (gave up: let what was issued complete before the memory goes)
        atomicExch(c.status, ERR_WAIT_MMA);
        tc_commit(drain);
        (void)mbar_wait(drain, 0);
      }
    }
    __syncwarp();
    tc_fence_before();
    } else {
      meet();                                                     // (behind regs_down: the softmax warps wait for those registers)
    }
  }
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after();
    tmem_dealloc<1>(*slot_at, 512);
  }
}

template <int D>
int chunk_launch(const Chunk8& c, cudaStream_t st_) {
  static std::atomic<uint64_t> set{0};                            // devices whose limit has been raised
  int dev = 0;
  if (int e = st::cuda_fail(cudaGetDevice(&dev), "st_kv8_chunk_attn: device")) return e;
  if (dev > 63 || !(set.load() >> dev & 1)) {
    if (int e = st::cuda_fail(cudaFuncSetAttribute(kv8_chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::BYTES),
                              "st_kv8_chunk_attn: shared memory attribute"))
      return e;
    if (dev <= 63) set.fetch_or(1ull << dev);
  }
  return st::launch("st_kv8_chunk_attn launch", kv8_chunk_kernel<D>, dim3((unsigned)((long long)c.slots * c.a.H * c.parts.splits)),
                    dim3(WARPS * 32), (size_t)Lay<D>::BYTES, st_, c);
}
}  // namespace

extern "C" int st_kv8_chunk_attn(const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv,
                                 const int8_t* exps, int64_t nblocks, int64_t Hkv, int64_t D, const int32_t* bt, int64_t bts,
                                 const int32_t* lens, const int32_t* starts, int64_t window, void* out, int64_t os, float* wo,
                                 float* wml, double scale, int64_t S, void* stream) {
  return st_kv8_chunk_attn_table(q, qs, T, Hq, cu, B, kv, exps, nblocks, Hkv, D, bt, bts, bts, lens, starts, window, out, os, wo, wml, scale,
                                 S, stream);
}

extern "C" int st_kv8_chunk_attn_table(const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv,
                                       const int8_t* exps, int64_t nblocks, int64_t Hkv, int64_t D, const int32_t* bt, int64_t btw,
                                       int64_t bts, const int32_t* lens, const int32_t* starts, int64_t window, void* out, int64_t os,
                                       float* wo, float* wml, double scale, int64_t S, void* stream) {
  Chunk8 c;
  if (int e = st::attn8_args(c.a, "st_kv8_chunk_attn", q, qs, T, Hq, cu, B, kv, exps, nblocks, Hkv, D, bt, btw, bts, lens, starts, window,
                             out, os, scale))
    return e;
  ST_REQUIRE(S >= 1 && S <= 1024, "st_kv8_chunk_attn: splits must be in [1, 1024]");
  ST_REQUIRE((wo && wml && st::aligned16(wo)) || st_kv8_attn_workspace_bytes(T, B, Hq, Hkv, D, S, 1) == 0,
             "st_kv8_chunk_attn: split workspace (wo, wml) missing or unaligned");
  if (T == 0 || B == 0) return 0;
  ST_REQUIRE(cu || T == B, "st_kv8_chunk_attn: without cu every sequence has one query");
  ST_REQUIRE(nblocks < (1ll << 31), "st_kv8_chunk_attn: too many pages");
  c.parts = {wo, wml, (int)S, 1};
  c.status = st::status_ptr();
  ST_REQUIRE(c.status != nullptr, "st_kv8_chunk_attn: no device status word");
  // 256-row tiles of all sequences: each may leave one unfilled
  const long long slots = T * (Hq / Hkv) / (2 * ROWS) + B;
  ST_REQUIRE(slots * Hkv * S < (1ll << 31) && T * (Hq / Hkv) < (1ll << 31), "st_kv8_chunk_attn: grid too large");
  c.slots = (int)slots;
  const cudaStream_t st_ = (cudaStream_t)stream;
  if (few_rows8(T, B, Hq / Hkv)) {
    c.parts.min_pages = 4;
    return st::rows8_attn("st_kv8_chunk_attn", c.a, c.parts, (int)D, st_);
  }
  const int e = D == 128 ? chunk_launch<128>(c, st_) : chunk_launch<64>(c, st_);
  if (e || S == 1) return e;
  return st::merge8("st_kv8_chunk_attn merge launch", c.a, c.parts, (int)D, st_);
}
