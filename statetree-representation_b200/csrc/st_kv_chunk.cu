// Causal attention of several query tokens per sequence straight over the lossless KV pages: prompts, their chunks, speculative tokens.
//     o = sum_j p_j v_j,  p = softmax_j(scale q . k_j),  j over [max(start, position - window + 1), position]
// Two kernels, by the rows (query token, head of the group) per sequence:
//   kv_chunk_kernel   many rows: tcgen05, 256 rows a CTA, 128 keys a step; pages are decoded into BF16 operand tiles in shared memory
//   kv_rows_kernel    few rows: mma.sync, 8 or 16 rows a CTA, a warp per page: the decode attention (kv_attn_kernel) with rows as columns
// Keys and values are exactly what was appended (BF16), scores are fp32 sums of exact products.  P is rounded to BF16 for the matrix
// instruction that V's type asks for: 2^-9 of each probability at most, of either sign (its sum is of the fp32 values), below the rounding
// of the output.  Everything else is fp32.
//
// Keys outside [start, len) of a sequence weigh nothing whatever their rows hold: scores are replaced, not shifted, and V's rows are zeroed
// on the way into the operands (a probability of 0 times an infinity would be NaN).
#include <float.h>
#include <math.h>

#include <atomic>

#include "../../include/statetree_b200.h"
#include "st_chunk_tc.cuh"
#include "st_host.h"
#include "st_kv.cuh"

namespace {
using namespace st;

// Warps of kv_chunk_kernel: eight of softmax, eight converters (a page of a key tile each), one that issues the MMAs, three producers
constexpr int W_MMA = W_CONV + TILE_PAGES, W_FETCH = W_MMA + 1, WARPS = W_MMA + 4, FETCHERS = WARPS - W_FETCH;
// registers of a warpgroup: 640 threads start with 96 each; 2 x 160 + 2 x 56 + 48 = 5 x 96
constexpr int R_START = 96, R_SOFTMAX = 160, R_CONV = 56, R_MMA = 48;
static_assert(2 * R_SOFTMAX + 2 * R_CONV + R_MMA <= 5 * R_START, "what the warpgroups take up is what the block starts with");
struct Pool { const uint32_t* at; int blocks; };
struct ChunkArgs { Attn8 a; Parts8 parts; Pool pool; int* status; int slots; };

// P is relative to a row's reference, the largest score seen up to RAISE before (base 2; BF16 has fp32's range: no lower bound is needed)
constexpr float RAISE = 8.f;

// ------------------------------------------------------------------------------------------------ many rows
// The division of the work, the hand-overs and the products are those of the attention over 8-bit pages (st_chunk_tc.cuh); what differs:
// there is no factor per page, and the converter warps decode records.  A warp takes one page of every key tile, its keys and then its values,
// from a slot of its own, which producer warps fill by bulk copies of 3200 bytes as soon as the records before are in registers (an issue
// takes some 270 cycles: one warp for all sixteen of a key tile would be the limit).  Decoded, a record is four mma A fragments: four stmatrix put it into the swizzled tile.  Its escapes are written over the tile, a lane an
// entry (patching the fragments instead takes a serial step an entry).
struct LayX : Tiles<HD> {
  static constexpr int RAW = Tiles<HD>::END, SLOT_BYTES = 2 * RKV;                                 // a slot per page of a key tile
  static constexpr int BARS = RAW + 8 * SLOT_BYTES, NBARS = ChunkBars::COUNT + 16, SLOT = BARS + NBARS * 8;
  static constexpr int BYTES = SLOT + 16 + 1024;
};

// A list of entries of a page's two units, half a warp for each unit, `listed` of them.  They ascend unless a row has been appended again in
// place: does one not?
__device__ __forceinline__ bool out_of_order(uint32_t entry, bool listed, int lane) {
  const uint32_t key = listed ? entry & 1023u : 0u, before = __shfl_up_sync(FULL, key, 1, 16);
  return __any_sync(FULL, listed && (lane & 15) > 0 && key <= before);
}
// the entries over the units' tile; `one_by_one`: so that the later entry of an element stands
__device__ __forceinline__ void put_entries(uint8_t* tile, uint32_t entry, bool wanted, bool one_by_one, int lane) {
  const int row = (int)((entry >> 6) & 15u), col = (int)(entry & 63u);
  uint16_t* const to = reinterpret_cast<uint16_t*>(tile + (lane >> 4) * LayX::HALF + row * 128 + ((((col >> 3) ^ (row & 7)) << 4) | (col & 7) * 2));
#pragma unroll 1
  for (int i = one_by_one ? 0 : 15; i < 16; ++i) {
    if (wanted && (!one_by_one || (lane & 15) == i)) *to = (uint16_t)(entry >> 16);
    __syncwarp();
  }
}

__global__ void __launch_bounds__(WARPS * 32, 1) kv_chunk_kernel(const ChunkArgs c) {
  constexpr int D = HD;
  using L = LayX;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  const ChunkBars b(reinterpret_cast<uint64_t*>(smem + L::BARS));
  uint64_t *const raw = b.rest, *const rempty = raw + 8;           // of every slot: filled, in registers
  uint32_t* const slot_at = reinterpret_cast<uint32_t*>(smem + L::SLOT);
  const Attn8& a = c.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.Hq / a.H;
  pdl_wait();
  pdl_launch_dependents();
  Work w;
  if (!chunk_work(a, c.parts.splits, c.slots, G, lane, w)) return;
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
    const int hi = live ? min(pos, a.table_width * PAGE - 1) : 0x7FFFFFFF, lo = !live ? 0 : window_from(a.window, pos, w.lo0);
    const bool any = __any_sync(FULL, live);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    // ---- the warp's 32 rows of q: sixteen lanes read a row
    if (count > 0) {
      const long long mine = live ? (long long)(w.first + token) * a.q_stride + (long long)hq * D : -1;
      const int col = lane & 15;
      uint8_t* const rows = smem + L::Q + t * L::TILE + (warp & 3) * (32 * 128) + (col >> 3) * L::HALF;
      uint4 u[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const long long from = __shfl_sync(FULL, mine, 2 * i + (lane >> 4));
        u[i] = from >= 0 ? *reinterpret_cast<const uint4*>(a.q + from + 8 * col) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 2 * i + (lane >> 4);
        *reinterpret_cast<uint4*>(rows + r * 128 + (((col & 7) ^ (r & 7)) << 4)) = u[i];
      }
      fence_proxy_async();
    }
    meet();
    const uint32_t tmem = *slot_at + ((uint32_t)((warp & 3) * 32) << 16), ts = tmem + t * 128, to = tmem + 256 + t * D;
    // The second row tile begins when the first has its first P: from then on each has the special function units to itself while the
    // other's products run.  (A barrier of its own, which completes once: the first tile's softmax does not wait for this one's, so that
    // it could complete a phase of `pfull` and the next before a warp here has looked)
    if (t == 1 && count > 0 && w.count0 > 0) ok = mbar_wait(b.begin1, 0);
    for (int j = 0; ok && j < count; ++j) {
      if (!mbar_wait_look(b.sfull + t, (uint32_t)j & 1u)) { ok = false; break; }
      tc_fence_after();
      if (any) {
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
        float x = __uint_as_float(v[0]), y = __uint_as_float(v[1]);
#pragma unroll
        for (int k = 2; k < KEYS - 2; k += 4) {
          x = max3(x, __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
          y = max3(y, __uint_as_float(v[k + 2]), __uint_as_float(v[k + 3]));
        }
        x = max3(x, __uint_as_float(v[KEYS - 2]), __uint_as_float(v[KEYS - 1]));
        const float top = fmaxf(x, y) * a.scale_log2;
        if (__any_sync(FULL, top > m + RAISE)) {
          const float up = fmaxf(m, top), f = up == m ? 1.f : ex2(m - up);
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
        const float ref = m == -INFINITY ? 0.f : -m;
        const uint64_t by2 = pair2(a.scale_log2, a.scale_log2), add2 = pair2(ref, ref);
        uint64_t sum = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float x0, x1;
            unpair2(fma2(pair2(__uint_as_float(v[32 * q + k]), __uint_as_float(v[32 * q + k + 1])), by2, add2), x0, x1);
            x0 = ex2(x0);
            x1 = ex2(x1);
            sum = add2f(sum, pair2(x0, x1));
            pk[k / 2] = pack_bf16(x0, x1);
          }
          tm_st16(ts + 16 * q, pk);
          if (q == 1) {                                           // the product with the first 64 keys need not wait for the others
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b.pfull + t);
          }
        }
        float s0, s1;
        unpair2(sum, s0, s1);
        l += s0 + s1;
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (!any) mbar_arrive(b.pfull + t);
        mbar_arrive(b.pfull + 2 + t);
        if (t == 0 && j == 0) mbar_arrive(b.begin1);
      }
    }
    if (ok && count > 0) ok = mbar_wait(b.ofull + t, 0);
    if (!ok && lane == 0) atomicExch(c.status, ERR_WAIT_ACC);
    // ---- out.  (a wait that ran out leaves the rows unwritten)
    if (ok && any) chunk_store<D>(a, c.parts, w, smem, t, warp, lane, live, token, hq, count, to, m, l);
    tc_fence_before();
  } else if (warp < W_MMA) {
    regs_down<R_CONV>();
    // ---------------------------------------------------------------- converters: records -> operand tiles
    const int cw = warp - W_CONV;
    const uint8_t* const unit = smem + L::RAW + cw * L::SLOT_BYTES;
    meet();
    // where this lane's rows of the four 8 x 8 blocks of a k-step go: row lane % 16, columns 8 (lane / 16) on
    const int at_row = (lane & 15) * 128, at_col = lane >> 4;
    bool ok = true;
    for (int j = 0; ok && j < tiles; ++j) {
      const int s = j & 1;
#pragma unroll 1                                                  // (twice the code costs more, in instruction fetches, than it saves)
      for (int kvi = 0; kvi < 2; ++kvi) {
        ok = mbar_wait_look(raw + cw, (uint32_t)kvi);            // (two phases a tile)
        if (!ok) break;
        const bool there = (w.first_tile + j) * TILE_PAGES + cw < end_page;
        uint32_t A[2][4][4], heads = 0u, head = 0u, ent = 0u, word = 0u;       // head, ent, word: of the lane's unit, lane / 16
        bool listed = false, odd = false;
        if (there) {
          RecRegs r[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            r[h] = load_rec_shared(unit + h * RKV, lane);
            heads |= *reinterpret_cast<const uint32_t*>(unit + h * RKV + REC);
          }
          const uint8_t* const tail = unit + (lane >> 4) * RKV + REC;
          head = *reinterpret_cast<const uint32_t*>(tail);
          ent = *reinterpret_cast<const uint32_t*>(tail + 4 + 4 * min(lane & 15, NSLOT - 1));
          __syncwarp();
          if (lane == 0) mbar_arrive(rempty + cw);
          listed = (lane & 15) < (int)min(head & 15u, (uint32_t)NSLOT);
          odd = out_of_order(ent, listed, lane);
          if ((head & 16u) && (int)(head >> 8) < c.pool.blocks)  // (requested here, looked at behind the decoding)
            word = __ldg(c.pool.at + (size_t)(head >> 8) * 16 + (lane & 15));
          decode_frag(r[0], A[0]);
          decode_frag(r[1], A[1]);
        } else {                                                // (a page that is not there: zeros)
          if (lane == 0) mbar_arrive(rempty + cw);
#pragma unroll
          for (int i = 0; i < 32; ++i) A[i >> 4][(i >> 2) & 3][i & 3] = 0u;
        }
        const int first = (w.first_tile + j) * KEYS + cw * PAGE;                  // position of the page's first token
        const bool edge = kvi && (first < w.start || first + PAGE > w.len);
        if (edge) {
          const int pos = first + (lane >> 2);
          const bool x0 = pos >= w.start && pos < w.len, x8 = pos + 8 >= w.start && pos + 8 < w.len;
#pragma unroll
          for (int i = 0; i < 32; ++i) A[i >> 4][(i >> 2) & 3][i & 3] = ((i & 1) ? x8 : x0) ? A[i >> 4][(i >> 2) & 3][i & 3] : 0u;
        }
        // K's stage is free when the scores of tile j - 2 are, V's when its products are: see the commits of the MMA loop
        const int e = kvi ? j - 1 : j - 2;
        if (j > 1) ok = mbar_wait_look(b.empty + (e & 1), (uint32_t)(e >> 1) & 1u);
        if (!ok) break;
        uint8_t* const tile = smem + (kvi ? L::V : L::K) + s * L::TILE + cw * (PAGE * 128);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t to = smem_addr(tile + h * L::HALF + at_row);
#pragma unroll
          for (int i = 0; i < 4; ++i) stmatrix_x4(to + (((2 * i + at_col) ^ (lane & 7)) << 4), A[h][i][0], A[h][i][1], A[h][i][2], A[h][i][3]);
        }
        if ((heads & 31u) != 0u) {                              // (the same in every lane)
          __syncwarp();
          int blk = (head & 16u) ? (int)(head >> 8) : -1;
#pragma unroll 1
          for (int hops = 0; hops < 4096; ++hops) {
            const int pos = first + (int)((ent >> 6) & 15u);
            put_entries(tile, ent, listed && (!edge || (pos >= w.start && pos < w.len)), odd, lane);
            const bool more = blk >= 0 && blk < c.pool.blocks;
            if ((heads & 16u) == 0u || !__any_sync(FULL, more)) break;
            if (hops > 0 && more) word = __ldg(c.pool.at + (size_t)blk * 16 + (lane & 15));
            const uint32_t w0 = __shfl_sync(FULL, word, 0, 16);
            ent = word;
            listed = more && (lane & 15) > 0 && (lane & 15) <= (int)min(w0 & 0xFFu, (uint32_t)XSLOT);
            odd = out_of_order(ent, listed, lane);
            blk = more ? (int)(w0 >> 8) - 1 : -1;
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive((kvi ? b.vfull : b.kfull) + s);
      }
    }
    if (!ok && lane == 0) atomicExch(c.status, ERR_WAIT_EMPTY);
  } else {
    regs_down<R_MMA>();
    if (warp == W_MMA) {
      // -------------------------------------------------------------- MMAs.  V is read as it lies (dims contiguous: MN-major)
      meet();
      if (elect_one())
        issue_mmas<D, mma_idesc(128, KEYS), mma_idesc(128, D) | 1u << 16>(smem, b, *slot_at, tiles, w.count0, w.count1, c.status);
      __syncwarp();
      tc_fence_before();
    } else {
      // -------------------------------------------------------------- producers: pages -> slots, a key tile's keys, then its values; warp f
      // brings pages f, f + 3, f + 6 of the eight
      const int f = warp - W_FETCH;
      const uint8_t* const head_pages = a.kv + (size_t)w.h * PAGE_BYTES;
      const size_t page_step = (size_t)a.H * PAGE_BYTES;
      const int* const table = a.table + (long long)w.b * a.table_stride;
      // lane l holds the entry of page l % 8 of the (l / 8)-th of four key tiles; -1 = there is no such page
      auto entry = [&](int j) {
        const int t = j + (lane >> 3), p = (w.first_tile + t) * TILE_PAGES + (lane & 7);
        if (t >= tiles || p >= end_page) return -1;
        const int e = __ldg(table + p);
        return e < 0 ? 0 : (int)min((long long)e, a.nblocks - 1);
      };
      if (lane < 8 && lane % FETCHERS == f) {
        mbar_init(raw + lane, 1);
        mbar_init(rempty + lane, 1);
        fence_barrier_init();
      }
      __syncwarp();
      int now = entry(0), next = -1;
      auto fetch = [&](int i, int kvi, int e) {                   // keys or values of page i of a tile
        if (elect_one()) {
          mbar_expect_tx(raw + i, e >= 0 ? (uint32_t)L::SLOT_BYTES : 0u);
          if (e >= 0) bulk_g2s(smem + L::RAW + i * L::SLOT_BYTES, head_pages + e * page_step + kvi * L::SLOT_BYTES, L::SLOT_BYTES, raw + i, keep);
        }
        __syncwarp();
      };
      if (tiles > 0)
        for (int i = f; i < 8; i += FETCHERS) fetch(i, 0, __shfl_sync(FULL, now, i));
      meet();
      bool ok = true;
      for (int j = 0; ok && j < tiles; ++j) {
        if ((j & 3) == 0) next = entry(j + 4);
#pragma unroll 1
        for (int kvi = j == 0; ok && kvi < 2; ++kvi) {
          const int n = 2 * j + kvi;                              // fetches into every slot before this round
          int i = f;
          for (; i < 8; i += FETCHERS) {
            ok = mbar_wait_look(rempty + i, (uint32_t)(n - 1) & 1u);
            if (!ok) break;
            fetch(i, kvi, __shfl_sync(FULL, now, 8 * (j & 3) + i));
          }
          if (!ok) {                                              // copies in flight land before the CTA ends: the last of every slot
            if (lane == 0) atomicExch(c.status, ERR_WAIT_EMPTY);
            for (int k = f; k < 8; k += FETCHERS) (void)mbar_wait(raw + k, (uint32_t)(k < i ? n : n - 1) & 1u);
          }
        }
        if ((j & 3) == 3) now = next;
      }
    }
  }
  __syncthreads();
  if (warp == W_MMA) {
    tc_fence_after();
    tmem_dealloc<1>(*slot_at, 512);
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// Rows (query, head) of a sequence on the 8-wide N side, NT times, tokens and dims on the M side; the pages of a CTA go round-robin to
// its warps, each with a ring of its own (kv_attn_kernel).  A page's records are decoded once for all of the CTA's rows: with sixteen rows a
// CTA of two column blocks does half of the decoding of two.
template <int NW, int STG, int NT>
__global__ void __launch_bounds__(NW * 32, (NT == 1 ? 16 : 12) / NW) kv_rows_kernel(const ChunkArgs c) {
  constexpr int COLS = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + (size_t)NW * STG * PAGE_BYTES);
  uint2* const sq = reinterpret_cast<uint2*>(bars + NW * STG);    // [column block][k-step][lane]: q as B fragments
  const Attn8& a = c.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, G = a.Hq / a.H;
  const int split = blockIdx.x % c.parts.splits, rest = blockIdx.x / c.parts.splits, kvh = rest % a.H;
  uint8_t* const ring = smem + (size_t)warp * STG * PAGE_BYTES;
  uint64_t* const bar = bars + warp * STG;
  if (lane == 0) {
    for (int s = 0; s < STG; ++s) mbar_init(bar + s, 1);
    fence_barrier_init();
  }
  const uint64_t keep = policy_evict_last();                      // (other rows read the same pages)
  pdl_wait();
  pdl_launch_dependents();
  Rows8 w;
  if (!find_rows<COLS>(a, G, rest / a.H, lane, w)) return;
  const int pos0 = w.len - w.n;
  const int p0 = pos0 + w.row0 / G, p1 = pos0 + (w.row0 + w.rows - 1) / G;                   // first and last position of the rows
  const int lo = window_from(a.window, p0, w.start), all_lo = window_from(a.window, p1, w.start);       // (every row sees [all_lo, p0])
  // ---- this warp's pages
  const int first_page = lo / PAGE, end_page = p1 >= lo ? min(p1 / PAGE + 1, a.table_width) : 0;
  const int per = max(c.parts.min_pages, (end_page - first_page + c.parts.splits - 1) / c.parts.splits);
  const int lo_page = first_page + split * per, hi_page = min(end_page, lo_page + per);
  const int my_first = lo_page + warp, my_count = hi_page > my_first ? (hi_page - my_first + NW - 1) / NW : 0;
  __syncwarp();
  const int* const my_table = a.table + (long long)w.b * a.table_stride + my_first;
  int entries = 0;
  auto fetch = [&](int i) {                                       // this warp's i-th page -> stage i % STG (whole warp, i in order)
    if ((i & 31) == 0) entries = i + lane < my_count ? __ldg(my_table + (i + lane) * NW) : 0;
    long long blk = __shfl_sync(FULL, entries, i & 31);
    blk = blk < 0 ? 0 : (blk >= a.nblocks ? a.nblocks - 1 : blk);
    if (elect_one()) {
      mbar_expect_tx(bar + i % STG, PAGE_BYTES);
      bulk_g2s(ring + (size_t)(i % STG) * PAGE_BYTES, a.kv + ((size_t)blk * a.H + kvh) * PAGE_BYTES, PAGE_BYTES, bar + i % STG, keep);
    }
    __syncwarp();
  };
  for (int i = 0; i < min(my_count, STG); ++i) fetch(i);
  // ---- q: column g of block nt, dims 16 ks + 2t, + 1 and 16 ks + 8 + 2t, + 1
  for (int i = warp; i < NT * 8; i += NW) {
    const int r = (i >> 3) * 8 + g, ks = i & 7;
    uint2 v = make_uint2(0u, 0u);
    if (r < w.rows) {
      const uint16_t* const row = a.q + (long long)(w.first + (w.row0 + r) / G) * a.q_stride + (kvh * G + (w.row0 + r) % G) * HD + 16 * ks + 2 * t;
      v = make_uint2(*reinterpret_cast<const uint32_t*>(row), *reinterpret_cast<const uint32_t*>(row + 8));
    }
    sq[i * 32 + lane] = v;
  }
  __syncthreads();
  // ---- running state of the lane's columns 8 nt + 2t + i; a column that is none sees nothing
  int hi_c[NT][2];
  float m[NT][2], l[NT][2], acc[NT][8][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * nt + 2 * t + i;
      hi_c[nt][i] = r < w.rows ? pos0 + (w.row0 + r) / G : -0x40000000;
      m[nt][i] = -INFINITY;
      l[nt][i] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[nt][k][2 * i] = acc[nt][k][2 * i + 1] = 0.f;
    }
  bool gave_up = false;
  for (int i = 0; i < my_count; ++i) {
    const int s = i % STG, tok = (my_first + i * NW) * PAGE;
    if (!mbar_wait(bar + s, (uint32_t)(i / STG) & 1u)) {
      if (lane == 0) atomicExch(c.status, ERR_WAIT_FULL);
      for (int k = i + 1; k < min(my_count, i + STG); ++k) (void)mbar_wait(bar + k % STG, (uint32_t)(k / STG) & 1u);   // (let what is in flight land)
      gave_up = true;
      break;
    }
    const uint8_t* const pg = ring + (size_t)s * PAGE_BYTES;
    // ---- S^T = K Q^T
    float sc[NT][4];
    {
      uint32_t R[2][4][4];
      units_to_frag(pg, c.pool.at, c.pool.blocks, lane, R);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) sc[nt][k] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint2 x = sq[(nt * 8 + ks) * 32 + lane], y = sq[(nt * 8 + 4 + ks) * 32 + lane];
          mma_bf16(sc[nt], R[0][ks], x.x, x.y);
          mma_bf16(sd, R[1][ks], y.x, y.y);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) sc[nt][k] = (sc[nt][k] + sd[k]) * a.scale_log2;
      }
    }
    if (tok < all_lo || tok + PAGE - 1 > p0 || w.rows < COLS) {   // some row does not see all of the page
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int p = hi_c[nt][k & 1], key = tok + g + 4 * (k & 2);
          if (key > p || key < window_from(a.window, p, w.start)) sc[nt][k] = -INFINITY;
        }
    }
    float top[NT][2];
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        top[nt][k] = fmaxf(sc[nt][k], sc[nt][k + 2]);
        raise = raise || top[nt][k] > m[nt][k] + RAISE;
      }
    if (__any_sync(FULL, raise)) {                                // bring the references to the page's true maxima, the sums along
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float up = fmaxf(m[nt][k], max_over_rows(top[nt][k])), f = up == m[nt][k] ? 1.f : ex2(m[nt][k] - up);
          m[nt][k] = up;
          l[nt][k] *= f;
#pragma unroll
          for (int q = 0; q < 8; ++q) { acc[nt][q][k] *= f; acc[nt][q][k + 2] *= f; }
        }
    }
    // ---- P^T as the B operand: the score fragment is [token][row]; transposed it is [row g][tokens 2t, 2t + 1].  As high part and
    // residual, like the decode attention: the matrix unit has room
    uint32_t pb[NT][2], rb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float r0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], r1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float x = ex2(sc[nt][2 * k] - r0), y = ex2(sc[nt][2 * k + 1] - r1);
        l[nt][0] += x;
        l[nt][1] += y;
        const uint32_t hi = pack_bf16(x, y);
        pb[nt][k] = movmatrix_t(hi);
        rb[nt][k] = movmatrix_t(pack_bf16(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xFFFF0000u)));
      }
    }
    // ---- O^T += V^T P^T
    {
      uint32_t R[2][4][4];
      units_to_frag(pg + 2 * RKV, c.pool.at, c.pool.blocks, lane, R);
      if (tok < w.start || tok + PAGE > w.len) {
        const bool x0 = tok + g >= w.start && tok + g < w.len, x8 = tok + 8 + g >= w.start && tok + 8 + g < w.len;
#pragma unroll
        for (int k = 0; k < 32; ++k) R[k >> 4][(k >> 2) & 3][k & 3] = ((k & 1) ? x8 : x0) ? R[k >> 4][(k >> 2) & 3][k & 3] : 0u;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          // 8 x 8 blocks of the record (tokens x dims) transposed: rows become dims, the k index becomes tokens
          const uint32_t a0 = movmatrix_t(R[half][ks][0]), a1 = movmatrix_t(R[half][ks][2]);
          const uint32_t a2 = movmatrix_t(R[half][ks][1]), a3 = movmatrix_t(R[half][ks][3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16_r(acc[nt][half * 4 + ks], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            mma_bf16_r(acc[nt][half * 4 + ks], a0, a1, a2, a3, rb[nt][0], rb[nt][1]);
          }
        }
    }
    __syncwarp();                                  // every lane has read this stage
    if (i + STG < my_count) {
      fence_proxy_async();
      fetch(i + STG);
    }
  }
  // ---- the warps' parts join: each parks (O^T, m, l) of its rows where its ring was
  __syncthreads();
  float* const park = reinterpret_cast<float*>(smem);
  constexpr int ROW = HD + 2, PER_WARP = COLS * ROW;
  static_assert(PER_WARP * 4 <= STG * PAGE_BYTES, "parked partials must fit in the ring");
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float* const mine = park + warp * PER_WARP + (8 * nt + 2 * t + k) * ROW;
#pragma unroll
      for (int q = 0; q < 8; ++q) { mine[16 * q + g] = acc[nt][q][k]; mine[16 * q + 8 + g] = acc[nt][q][k + 2]; }
      const float sum = sum_over_rows(l[nt][k]);
      if (g == 0) { mine[HD] = gave_up ? -INFINITY : m[nt][k]; mine[HD + 1] = gave_up ? 0.f : sum; }
    }
  __syncthreads();
  for (int e = threadIdx.x; e < w.rows * HD; e += NW * 32) {
    const int r = e / HD, d = e % HD;
    float top = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, park[i * PER_WARP + r * ROW + HD]);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float* const p = park + i * PER_WARP + r * ROW;
      if (p[HD] == -INFINITY && p[HD + 1] == 0.f) continue;       // a warp that has seen nothing
      const float f = p[HD] == top ? 1.f : ex2(p[HD] - top);
      den = fmaf(f, p[HD + 1], den);
      num = fmaf(f, p[d], num);
    }
    const long long tk = w.first + (w.row0 + r) / G;
    const int hq = kvh * G + (w.row0 + r) % G;
    if (c.parts.splits == 1) {
      const __nv_bfloat16 v = __float2bfloat16_rn(den > 0.f ? num / den : den);
      a.out[tk * a.out_stride + (long long)hq * HD + d] = *reinterpret_cast<const uint16_t*>(&v);
    } else {
      const long long ix = (tk * a.Hq + hq) * c.parts.splits + split;
      c.parts.o[ix * HD + d] = num;
      if (d == 0) { c.parts.ml[ix * 2] = top; c.parts.ml[ix * 2 + 1] = den; }
    }
  }
}

template <typename Kernel>
int opt_in(Kernel* kernel, int bytes, std::atomic<uint64_t>& set) {
  int dev = 0;                                                    // (set: devices whose limit has been raised)
  if (int e = st::cuda_fail(cudaGetDevice(&dev), "st_kv_chunk_attn: device")) return e;
  if (dev <= 63 && (set.load() >> dev & 1)) return 0;
  if (int e = st::cuda_fail(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "st_kv_chunk_attn: shared memory attribute"))
    return e;
  if (dev <= 63) set.fetch_or(1ull << dev);
  return 0;
}
template <int NW, int NT>
int rows_launch(const ChunkArgs& c, long long ctas, cudaStream_t st_) {
  constexpr int STG = 2, BYTES = NW * STG * (PAGE_BYTES + 8) + NT * 8 * 32 * 8;
  static std::atomic<uint64_t> set{0};
  if (int e = opt_in(kv_rows_kernel<NW, STG, NT>, BYTES, set)) return e;
  return st::launch("st_kv_chunk_attn launch", kv_rows_kernel<NW, STG, NT>, dim3((unsigned)ctas), dim3(NW * 32), (size_t)BYTES, st_, c);
}
}  // namespace

extern "C" int64_t st_kv_chunk_attn_workspace_bytes(int64_t T, int64_t Hq, int64_t S) {
  return T <= 0 || Hq <= 0 || S <= 1 ? 0 : T * Hq * S * (st::HD + 2) * 4;
}

extern "C" int st_kv_chunk_attn(const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv, int64_t nblocks,
                                int64_t Hkv, const uint32_t* pool, int64_t P, const int32_t* bt, int64_t btw, int64_t bts,
                                const int32_t* lens, const int32_t* starts, int64_t window, void* out, int64_t os, float* wo, float* wml,
                                double scale, int64_t S, void* stream) {
  const char* who = "st_kv_chunk_attn";
  ChunkArgs c;
  if (int e = st::attn8_args(c.a, who, q, qs, T, Hq, cu, B, kv, (const int8_t*)kv, nblocks, Hkv, HD, bt, btw, bts, lens, starts, window, out, os,
                             scale))
    return e;
  ST_REQUIRE(S >= 1 && S <= 1024, "%s: splits must be in [1, 1024]", who);
  if (T == 0 || B == 0) return 0;
  ST_REQUIRE(pool && P >= 0 && P < (1ll << 31), "%s: null pointer (pool)", who);
  ST_REQUIRE(S == 1 || (wo && wml && st::aligned16(wo)), "%s: split workspace (wo, wml) missing or unaligned", who);
  ST_REQUIRE(cu || T == B, "%s: without cu every sequence has one query", who);
  ST_REQUIRE(nblocks < (1ll << 31), "%s: too many pages", who);
  c.a.scale_log2 = fmaxf(c.a.scale_log2, FLT_MIN);                // (it multiplies the -inf of what a row does not see)
  c.parts = {wo, wml, (int)S, 4};
  c.pool = {pool, (int)P};
  c.status = st::status_ptr();
  ST_REQUIRE(c.status != nullptr, "%s: no device status word", who);
  const long long G = Hq / Hkv;
  ST_REQUIRE(T * G < (1ll << 31), "%s: too large", who);
  const cudaStream_t st_ = (cudaStream_t)stream;
  auto ctas_of = [&](long long rows) { return (T * G / rows + B) * Hkv * S; };                // (every sequence may leave a tile unfilled)
  int e;
  if (st::few_rows8(T, B, G)) {
    const bool two = T * G > 8 * B;
    const long long ctas = ctas_of(two ? 16 : 8);
    ST_REQUIRE(ctas < (1ll << 31), "%s: grid too large", who);
    // (an SM holds sixteen warps of eight rows, as CTAs of four or two of eight, or twelve of sixteen rows: three CTAs of four, one of eight)
    e = two ? (ctas <= st::sm_count() ? rows_launch<8, 2>(c, ctas, st_) : rows_launch<4, 2>(c, ctas, st_))
            : (ctas <= 2ll * st::sm_count() ? rows_launch<8, 1>(c, ctas, st_) : rows_launch<4, 1>(c, ctas, st_));
  } else {
    static std::atomic<uint64_t> set{0};
    const long long ctas = ctas_of(2 * ROWS);
    ST_REQUIRE(ctas < (1ll << 31), "%s: grid too large", who);
    c.slots = (int)(ctas / Hkv / S);
    if (int r = opt_in(kv_chunk_kernel, LayX::BYTES, set)) return r;
    e = st::launch("st_kv_chunk_attn launch", kv_chunk_kernel, dim3((unsigned)ctas), dim3(WARPS * 32), (size_t)LayX::BYTES, st_, c);
  }
  if (e || S == 1) return e;
  return st::merge8("st_kv_chunk_attn merge launch", c.a, c.parts, HD, st_);
}
