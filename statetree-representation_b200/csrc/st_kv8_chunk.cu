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
#include "st_chunk_tc.cuh"

namespace {
using namespace st;

constexpr int W_MMA = 12, WARPS = 16;                             // (four converter warps; 13 .. 15 only lend registers)
// registers of a warpgroup: 512 threads start with 128 each (64 K in all, the SM's); 2 x 184 + 96 + 48 = 4 x 128
constexpr int R_SOFTMAX = 184, R_CONV = 96, R_MMA = 48;
constexpr int CRING = 4;                                          // page factors of so many key tiles are kept

template <int D>
struct Lay : Tiles<D> {                                           // shared memory
  static constexpr int RAW = Tiles<D>::END, UNIT = PAGE * D;      // codes of one key tile: its keys, its values
  static constexpr int F = RAW + 2 * TILE_PAGES * UNIT, BARS = F + CRING * TILE_PAGES * 3 * 4;
  static constexpr int NBARS = ChunkBars::COUNT + 8, SLOT = BARS + NBARS * 8;
  // (more than half of an SM's shared memory: one CTA per SM, which holds all of its tensor memory)
  static constexpr int BYTES = (SLOT + 16 > 120 * 1024 ? SLOT + 16 : 120 * 1024) + 1024;
};

struct Chunk8 { Attn8 a; Parts8 parts; int* status; int slots; };

template <int D>
__global__ void __launch_bounds__(WARPS * 32, 1) kv8_chunk_kernel(const Chunk8 c) {
  using L = Lay<D>;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  const ChunkBars b(reinterpret_cast<uint64_t*>(smem + L::BARS));
  uint64_t *const begin1 = b.begin1, *const kfull = b.kfull, *const vfull = b.vfull, *const sfull = b.sfull, *const pfull = b.pfull,
           *const ofull = b.ofull, *const empty = b.empty, *const raw = b.rest;                  // raw: [converter warp][keys, values]
  uint32_t* const slot_at = reinterpret_cast<uint32_t*>(smem + L::SLOT);
  const Attn8& a = c.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.Hq / a.H;
  pdl_wait();
  pdl_launch_dependents();

  Work w;
  if (!chunk_work<2 * ROWS>(a, blockIdx.x / c.parts.splits, blockIdx.x % c.parts.splits, c.parts.splits, c.slots, G, lane, w)) return;
  const int tiles = max(w.count0, w.count1);
  // (pages behind the last key of the sequence, or behind its row of the table, may not exist: no key of theirs is seen)
  const int end_page = min((w.pos0 + w.n - 1) / PAGE + 1, a.table_width);
  const uint64_t keep = policy_evict_last();                      // other row tiles of the sequence read the same pages

  if (warp == W_MMA) {
    if (elect_one()) b.init(W_MMA - W_CONV);
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
    if (ok && any) chunk_store<D, false>(a, c.parts, w, smem, t, warp, lane, live, token, hq, count, to, m, l);
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
    // ---------------------------------------------------------------- MMAs (mma_idesc's operands are BF16; FP16 is type 0)
    constexpr uint32_t FP16 = ~(1u << 7 | 1u << 10), IDESC_S = mma_idesc(128, KEYS) & FP16, IDESC_O = (mma_idesc(128, D) & FP16) | 1u << 16;
    meet();
    const uint32_t tmem = *slot_at;
    if (elect_one()) issue_mmas<D, IDESC_S, IDESC_O>(smem, b, tmem, tiles, w.count0, w.count1, c.status);
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
