// Causal attention of several query tokens per sequence straight over the lossless KV pages: prompts, their chunks, speculative tokens.
//     o = sum_j p_j v_j,  p = softmax_j(scale q . k_j),  j over [max(start, position - window + 1), position]
// on tcgen05, 128 keys a step; pages are decoded into BF16 operand tiles in shared memory.  Two forms, by the rows (query token, head of the
// group) per sequence: 256 rows a CTA, or (NARROW) 32.  The division of the work, the tensor-memory columns, the hand-overs and the products are
// those of the attention over 8-bit pages (st_chunk_tc.cuh, st_kv8_chunk.cu).
// Keys and values are exactly what was appended (BF16), scores are fp32 sums of exact products.  P is rounded to BF16, the type that the matrix
// instruction asks for beside V's: by 2^-8 of each probability at most, as the output's own rounding (its sum is of the fp32 values).
// Everything else is fp32.
//
// Keys outside [start, len) of a sequence weigh nothing whatever their rows hold: scores are replaced, not shifted, and V's rows are zeroed
// on the way into the operands (a probability of 0 times an infinity would be NaN).  Infinities and NaN of V at positions that the sequence has
// are zeroed there too, and the rows that see them get them on their way out: an infinity of either sign gives itself, both or NaN give NaN.
//
// Measured (32 query heads, 8 KV heads), us in a graph: 2048 queries behind 30000 tokens 1095-1120 = 0.94 PFLOP/s, a prompt of 4096 180, nine ragged
// chunks with windows (7 heads a KV head) 103; 8 x 4 queries over 2900 tokens 34.
// What bounds it.  A step of 256 rows takes 2.2 us, of which the MMAs fill 1.2: the chain scores -> softmax -> product of a row tile (with the
// conversion left out 1.9 us a step) and the converters, which share the issue slots with it (50 % used; 250 instructions a page's keys or
// values; escapes 0.2 us of the step).  A CTA costs some 12 us besides its steps (look-ups, q, filling and draining the two row tiles' chains,
// output).  32 rows: 1.45 us a step, 4.5 TB/s of pages from 128 SMs, and as much outside the steps as in them.
// Tried: four converter warps of two pages 1904 us (2048 behind 30000; they wait for one another's latencies), one producer warp 2241; P as high
// part and residual is a product more; a CTA of 8 or 16 rows on mma.sync, three to an SM, for few rows: 8 x 4 queries 37 us, 32 x 4 over 2000
// tokens 84 (here 70).
#include <float.h>
#include <math.h>

#include <atomic>

#include "../../include/statetree_b200.h"
#include "st_chunk_tc.cuh"
#include "st_host.h"

namespace {
using namespace st;

// Rows of a CTA of the narrow form, and per sequence (on the mean) up to which it is taken.  us with 32 / 256 rows a CTA, the better splits of
// each: 8 rows of 8 sequences of 2900 tokens 32.3 / 33.6, 32 rows 36.7 / 36.7, 64 rows 51.6 / 37.9; 32 rows of 32 sequences 75.5 / 80.9, 64 rows
// 143 / 82; 32 rows of one 21.9 / 20.0
constexpr int FEW = 32;
// Warps of kv_chunk_kernel: of softmax, of conversion (a page of a key tile each; NARROW: its keys or its values), one that issues the MMAs, three
// producers.  Registers of a warpgroup: what they take up together is at most what the block starts with, a multiple of 8 a thread
template <bool NARROW>
struct Roles {
  static constexpr int CONV = NARROW ? 4 : 8, CONVERTERS = NARROW ? 2 * TILE_PAGES : TILE_PAGES;
  static constexpr int MMA = CONV + CONVERTERS, FETCH = MMA + 1, WARPS = MMA + 4, FETCHERS = WARPS - FETCH, GROUPS = WARPS / 4;
  static constexpr int R_START = 65536 / (WARPS * 32) / 8 * 8, R_SOFTMAX = NARROW ? 112 : 152, R_CONV = NARROW ? 80 : 72, R_MMA = 32;
  static_assert(CONV / 4 * R_SOFTMAX + CONVERTERS / 4 * R_CONV + R_MMA <= GROUPS * R_START, "more registers than there are");
};
struct Pool { const uint32_t* at; int blocks; };
struct ChunkArgs { Attn8 a; Parts8 parts; Pool pool; int* status; int slots, whole; };           // whole: units that are not split, the first ones

// P is relative to a row's reference, the largest score seen up to RAISE before (base 2; BF16 has fp32's range: no lower bound is needed)
constexpr float RAISE = 8.f;

// ------------------------------------------------------------------------------------------------ a page's keys or values -> a tile
// Two units (dims 0 .. 63, 64 .. 127) of raw bytes in shared memory become sixteen rows of two swizzled 128-byte halves, HALF bytes apart.  A
// decoded record is four mma A fragments: four stmatrix put it there.  Its escapes are written over the tile, a lane an entry and half a warp a
// unit (patching the fragments takes a serial step an entry: 2048 queries behind 30000 tokens 1.5 times as long).
struct Lists {                                     // of a page's two units: what a lane holds of the list of unit lane / 16
  uint32_t heads, head, entry, word;               // both units' headers together, its own, an entry, a word of its chain's first block
  bool listed, odd, beyond;                        // beyond: a value may be NaN or an infinity
};
// Entries ascend unless a row has been appended again in place: does one not?
__device__ __forceinline__ bool entry_out_of_order(uint32_t entry, bool listed, int lane) {
  const uint32_t key = listed ? entry & 1023u : 0u, before = __shfl_up_sync(FULL, key, 1, 16);
  return listed && (lane & 15) > 0 && key <= before;
}
__device__ __forceinline__ bool out_of_order(uint32_t entry, bool listed, int lane) { return __any_sync(FULL, entry_out_of_order(entry, listed, lane)); }
// is one of a lane's nodes, those of rows lane / 4 and 8 more of either unit, the largest exponent (NaN, infinities)
__device__ __forceinline__ bool node_beyond(const RecRegs (&r)[2]) {
  const uint32_t x = ~(r[0].nodes | r[1].nodes << 16);
  return ((x - 0x01010101u) & ~x & 0x80808080u) != 0u;
}
__device__ __forceinline__ void page_take(const uint8_t* unit, int lane, RecRegs (&r)[2], Lists& l) {
  l.heads = 0u;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    r[h] = load_rec_shared(unit + h * RKV, lane);
    l.heads |= *reinterpret_cast<const uint32_t*>(unit + h * RKV + REC);
  }
  const uint8_t* const tail = unit + (lane >> 4) * RKV + REC;
  l.head = *reinterpret_cast<const uint32_t*>(tail);
  l.entry = *reinterpret_cast<const uint32_t*>(tail + 4 + 4 * min(lane & 15, NSLOT - 1));
}
// (ahead of the decoding: the chain's block is looked at behind it)
template <bool NARROW>
__device__ __forceinline__ void page_lists(Lists& l, const RecRegs (&r)[2], const Pool& pool, bool values, int lane) {
  l.listed = (lane & 15) < (int)min(l.head & 15u, (uint32_t)NSLOT);
  if (NARROW) {                                    // (a warp has either keys or values: 8 x 4 queries 34.3 us, with the one vote 34.5)
    l.odd = out_of_order(l.entry, l.listed, lane);
    l.beyond = values && __any_sync(FULL, node_beyond(r));
  } else {
    const uint32_t flags = __reduce_or_sync(FULL, (entry_out_of_order(l.entry, l.listed, lane) ? 1u : 0u) | (node_beyond(r) ? 2u : 0u));
    l.odd = flags & 1u;
    l.beyond = values && (flags & 2u);
  }
  l.word = (l.head & 16u) && (int)(l.head >> 8) < pool.blocks ? __ldg(pool.at + (size_t)(l.head >> 8) * 16 + (lane & 15)) : 0u;
}
template <int HALF>
__device__ __forceinline__ void page_store(uint8_t* tile, const uint32_t (&A)[2][4][4], int lane) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {                    // (this lane names row lane % 16, columns 8 (lane / 16) on of every k-step)
    const uint32_t to = smem_addr(tile + h * HALF + (lane & 15) * 128);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      stmatrix_x4(to + (((2 * i + (lane >> 4)) ^ (lane & 7)) << 4), A[h][i][0], A[h][i][1], A[h][i][2], A[h][i][3]);
  }
}
// `edge`: only the rows of positions [start, len) (the page's first row is position `first`)
template <int HALF>
__device__ __forceinline__ void page_patch(uint8_t* tile, Lists& l, const Pool& pool, bool edge, int first, int start, int len, int lane) {
  if ((l.heads & 31u) == 0u) return;               // (the same in every lane)
  __syncwarp();
  auto put = [&](bool now) {
    const int row = (int)((l.entry >> 6) & 15u), col = (int)(l.entry & 63u), pos = first + row;
    if (now && l.listed && (!edge || (pos >= start && pos < len)))
      *reinterpret_cast<uint16_t*>(tile + (lane >> 4) * HALF + row * 128 + ((((col >> 3) ^ (row & 7)) << 4) | (col & 7) * 2)) = (uint16_t)(l.entry >> 16);
  };
  if (!l.odd && (l.heads & 16u) == 0u) {
    put(true);
    return;
  }
  int blk = (l.head & 16u) ? (int)(l.head >> 8) : -1;
#pragma unroll 1
  for (int hops = 0; hops < 4096; ++hops) {
#pragma unroll 1
    for (int i = l.odd ? 0 : 15; i < 16; ++i) {    // (out of order: one by one, so that the later entry of an element stands)
      put(!l.odd || (lane & 15) == i);
      __syncwarp();
    }
    const bool more = blk >= 0 && blk < pool.blocks;
    if (!__any_sync(FULL, more)) break;
    if (hops > 0 && more) l.word = __ldg(pool.at + (size_t)blk * 16 + (lane & 15));
    const uint32_t w0 = __shfl_sync(FULL, l.word, 0, 16);
    l.entry = l.word;
    l.listed = more && (lane & 15) > 0 && (lane & 15) <= (int)min(w0 & 0xFFu, (uint32_t)XSLOT);
    l.odd = out_of_order(l.entry, l.listed, lane);
    blk = more ? (int)(w0 >> 8) - 1 : -1;
  }
}
// What a CTA found among its values: first and last page with NaN or infinities, and for every dimension whether there is +inf or NaN, -inf or NaN
struct Beyond { int page0, page1; uint32_t plus[HD / 32], minus[HD / 32]; };
// A page's values that have the largest exponent (NaN, infinities): zeros instead, and a note.  Rare: such rows show in their nodes, which is all
// that the other pages pay (8 x 4 queries over 2900 tokens 34.3 us, 33.2 without the look and the note)
template <int HALF>
__device__ __forceinline__ void page_finite(uint8_t* tile, int page, Beyond* note, int lane) {
  bool found = false;
  __syncwarp();
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {                    // four rows of a half at a time, eight lanes a row
    uint4* const at = reinterpret_cast<uint4*>(tile + (i >> 2) * HALF) + (i & 3) * 32 + lane;
    const uint32_t w[4] = {at->x, at->y, at->z, at->w};
    uint32_t out[4], plus = 0u, minus = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      out[k] = w[k];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t bits = w[k] >> (16 * b);
        if ((bits & 0x7F80u) != 0x7F80u) continue;
        const bool nan = bits & 0x7Fu, less = bits & 0x8000u;
        plus |= nan || !less ? 1u << (2 * k + b) : 0u;
        minus |= nan || less ? 1u << (2 * k + b) : 0u;
        out[k] &= b ? 0xFFFFu : 0xFFFF0000u;
      }
    }
    if ((plus | minus) == 0u) continue;
    found = true;
    *at = make_uint4(out[0], out[1], out[2], out[3]);
    const int dim = 64 * (i >> 2) + 8 * ((lane & 7) ^ ((4 * (i & 3) + (lane >> 3)) & 7));
    atomicOr(&note->plus[dim >> 5], plus << (dim & 31));
    atomicOr(&note->minus[dim >> 5], minus << (dim & 31));
  }
  if (__any_sync(FULL, found) && lane == 0) {
    atomicMin(&note->page0, page);
    atomicMax(&note->page1, page);
  }
}
// rows of positions outside [start, len) to zero
__device__ __forceinline__ void page_edge(uint32_t (&A)[2][4][4], int first, int start, int len, int lane) {
  const int pos = first + (lane >> 2);
  const bool x0 = pos >= start && pos < len, x8 = pos + 8 >= start && pos + 8 < len;
#pragma unroll
  for (int i = 0; i < 32; ++i) A[i >> 4][(i >> 2) & 3][i & 3] = ((i & 1) ? x8 : x0) ? A[i >> 4][(i >> 2) & 3][i & 3] : 0u;
}

// ------------------------------------------------------------------------------------------------ the kernel
// A converter warp takes one page of every key tile, its keys and its values, from a slot of its own (a waiter must never be two phases of a
// barrier away: a slot has one producer and one consumer), which producer warps fill by bulk copies of 3200 bytes as soon as the records
// before are in registers (an issue takes some 270 cycles: one warp for all sixteen of a key tile would be the limit).
// NARROW: keys and values have slots of their own (the second set where the second row tile's q would be), so that a page's values come in while
// its keys are decoded: these pages are read once, from memory, not by many CTAs from L2.
struct Kept { int row0, rows, first, h, split, splits, b, pos0, start; Beyond beyond; };         // of Work, for the way out; splits: of this unit
struct LayX : Tiles<HD> {
  static constexpr int RAW = Tiles<HD>::END, SLOT_BYTES = 2 * RKV;                                 // a slot per page of a key tile
  static constexpr int BARS = RAW + 8 * SLOT_BYTES, NBARS = ChunkBars::COUNT + 34, SLOT = BARS + NBARS * 8, KEPT = SLOT + 16;
  static constexpr int BYTES = KEPT + sizeof(Kept) + 1024;
  static __device__ __forceinline__ int slot(int set, int page) { return (set ? Q + TILE : RAW) + page * SLOT_BYTES; }
};

// A bit for every one of 32 values of a row: it gets +inf, -inf; NaN is both
struct Seen {
  uint32_t p, n;
  __device__ __forceinline__ void to(uint32_t* v) const {
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      if (p >> k & 1u) v[k] = __float_as_uint(__uint_as_float(v[k]) + INFINITY);
      if (n >> k & 1u) v[k] = __float_as_uint(__uint_as_float(v[k]) - INFINITY);
    }
  }
};
// What values 32 q .. 32 q + 31 of this lane's row get: the infinities and NaN of the keys lo .. hi that it sees (`only` >= 0: of those in
// the only-th 32 of every 128), which lie in pages page0 .. page1.  Lane l looks at value 32 q + l of a key.  It ends when no row can get more
__device__ __forceinline__ Seen beyond_seen(const Attn8& a, const Pool& pool, const Kept& kept, int page0, int page1, int q, int lo, int hi, int only,
                                            int lane) {
  const int col = 32 * (q & 1) + lane;
  const uint8_t* const values = a.kv + (size_t)kept.h * PAGE_BYTES + (2 + (q >> 1)) * RKV;
  const size_t step = (size_t)a.H * PAGE_BYTES;
  const int* const table = a.table + (long long)kept.b * a.table_stride;
  const volatile Beyond& note = *const_cast<const volatile Beyond*>(&kept.beyond);
  const uint32_t all_p = __shfl_sync(FULL, note.plus[q], 0), all_n = __shfl_sync(FULL, note.minus[q], 0);
  uint32_t p = 0u, n = 0u;
#pragma unroll 1
  for (int p0 = page0; p0 <= page1; p0 += 32) {
    if (__all_sync(FULL, lo > hi || (p == all_p && n == all_n))) break;
    int e = 0;
    bool has = false;
    if (p0 + lane <= page1) {
      e = __ldg(table + p0 + lane);
      e = e < 0 ? 0 : (int)min((long long)e, a.nblocks - 1);
      const uint4 nodes = __ldg(reinterpret_cast<const uint4*>(values + e * step + 1536));
      has = ((__vcmpeq4(nodes.x, ~0u) | __vcmpeq4(nodes.y, ~0u)) | (__vcmpeq4(nodes.z, ~0u) | __vcmpeq4(nodes.w, ~0u))) != 0u;
    }
#pragma unroll 1
    for (uint32_t todo = __ballot_sync(FULL, has); todo; todo &= todo - 1) {
      const int i = __ffs(todo) - 1;
      const uint8_t* const unit = values + __shfl_sync(FULL, e, i) * step;
#pragma unroll 1
      for (uint32_t rows = __ballot_sync(FULL, lane < 16 && __ldg(unit + 1536 + 2 * (lane & 7) + (lane >> 3 & 1)) == 255); rows; rows &= rows - 1) {
        const int r = __ffs(rows) - 1, pos = (p0 + i) * PAGE + r;
        const bool sees = pos >= lo && pos <= hi && (only < 0 || (pos >> 5 & 3) == only);
        if (!__any_sync(FULL, sees)) continue;
        // column 16 s + 8 i + 2 t + b of row r: its leaf (mantissa << 1 | its neighbour's sign) and its state's nibble
        const int s = col >> 4, at = (r & 7) * 4 + (col & 7) / 2, two = (col >> 3 & 1) * 2;
        const uint8_t* const leaf = unit + (s >> 1) * 512 + at * 16 + ((s & 1) * 2 + (r >> 3)) * 4 + two;
        const uint32_t state = __ldg(unit + 1024 + at * 16 + s * 4 + two + (col & 1)) >> (4 * (r >> 3)) & 15u;
        uint32_t bits = state ? 0u : 0x7F80u | __ldg(leaf + (col & 1)) >> 1 | (__ldg(leaf + ((col & 1) ^ 1)) & 1u) << 15;
        uint32_t kp = 0u, kn = 0u;
        auto bits_of = [&] {
          const bool beyond = (bits & 0x7F80u) == 0x7F80u, nan = bits & 0x7Fu;
          kp = __ballot_sync(FULL, beyond && (nan || !(bits & 0x8000u)));
          kn = __ballot_sync(FULL, beyond && (nan || (bits & 0x8000u)));
        };
        bits_of();
        if (!__any_sync(FULL, sees && ((kp & ~p) | (kn & ~n)))) continue;
        // (an entry of a row that stood there before is what counts)
        auto look = [&](uint32_t entry) { if ((int)(entry & 1023u) == r * 64 + col) bits = entry >> 16; };
        const uint32_t head = __ldg(reinterpret_cast<const uint32_t*>(unit + REC));
        for (int k = 0; k < (int)min(head & 15u, (uint32_t)NSLOT); ++k) look(__ldg(reinterpret_cast<const uint32_t*>(unit + REC) + 1 + k));
        int blk = (head & 16u) ? (int)(head >> 8) : -1;
        for (int hops = 0; blk >= 0 && blk < pool.blocks && hops < 4096; ++hops) {
          const uint32_t w0 = __ldg(pool.at + (size_t)blk * 16);
          for (int k = 0; k < (int)min(w0 & 0xFFu, (uint32_t)XSLOT); ++k) look(__ldg(pool.at + (size_t)blk * 16 + 1 + k));
          blk = (int)(w0 >> 8) - 1;
        }
        bits_of();
        p |= sees ? kp : 0u;
        n |= sees ? kn : 0u;
      }
    }
  }
  return {p, n};
}

// NARROW: up to 32 rows, which stand four times in the first row tile, once for each of its softmax warps.  A warp forms P of 32 of a step's 128
// keys (zeros elsewhere), so that the chain scores -> softmax -> product is a quarter of the exponentials long, and its copy of the rows
// sums up those keys' values; here the four join.  (`ok` false: the rows stay unwritten)
template <class Last>
__device__ __forceinline__ void narrow_store(const Attn8& a, const Parts8& parts, const Work& w, uint8_t* const smem, int warp, int lane, bool ok,
                                             int count, uint32_t to, float m, float l, const Last last) {
  constexpr int ROW = HD + 4;                                     // (rows 33 x 16 bytes apart: no two lanes of eight in one bank)
  float* const park = reinterpret_cast<float*>(smem);             // [warp][row][ROW]: where q, K and V were
  float2* const ml = reinterpret_cast<float2*>(park + 4 * FEW * ROW);
  tc_fence_after();
  constexpr int AT_ONCE = std::is_same_v<Last, AsTheyAre> ? HD / 32 : 1;
#pragma unroll AT_ONCE
  for (int q = 0; q < HD / 32; ++q) {
    const auto more = last(q);
    uint32_t v[32];
    if (count > 0) {
      tm_ld32(to + 32 * q, v);
      tm_wait_ld<32>(v);
    }
#pragma unroll
    for (int k = 0; k < 32; ++k) v[k] = count > 0 && l != 0.f ? v[k] : 0u;
    more.to(v);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      *reinterpret_cast<uint4*>(park + (warp * FEW + lane) * ROW + 32 * q + 4 * k) = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
  }
  ml[warp * FEW + lane] = make_float2(l > 0.f || l != l ? m : -INFINITY, ok ? l : -1.f);      // (no sum is negative: a warp that gave up)
  named_bar_sync(1, 128);
  const int G = a.Hq / a.H;
  for (int r = warp; r < w.rows; r += 4) {
    float top = -INFINITY, den = 0.f;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    bool all = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i * FEW + r].x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = ml[i * FEW + r];
      all = all && x.y != -1.f;
      if (x.x == -INFINITY && x.y == 0.f) continue;               // a warp whose keys the row has not seen
      const float f = x.x == top ? 1.f : ex2(x.x - top);
      const float4 o = *reinterpret_cast<const float4*>(park + (i * FEW + r) * ROW + 4 * lane);
      den = fmaf(f, x.y, den);
      num.x = fmaf(f, o.x, num.x); num.y = fmaf(f, o.y, num.y); num.z = fmaf(f, o.z, num.z); num.w = fmaf(f, o.w, num.w);
    }
    if (!all) continue;
    const long long token = w.first + (w.row0 + r) / G;
    const int hq = w.h * G + (w.row0 + r) % G;
    if (parts.splits == 1) {
      const float inv = den > 0.f ? 1.f / den : den;
      *reinterpret_cast<uint2*>(a.out + token * a.out_stride + (long long)hq * HD + 4 * lane) =
          make_uint2(pack_bf16(num.x * inv, num.y * inv), pack_bf16(num.z * inv, num.w * inv));
    } else {
      const long long at = (token * a.Hq + hq) * parts.splits + w.split;
      *reinterpret_cast<float4*>(parts.o + at * HD + 4 * lane) = num;
      if (lane == 0) { parts.ml[at * 2] = top; parts.ml[at * 2 + 1] = den; }
    }
  }
}

template <bool NARROW>
__global__ void __launch_bounds__(Roles<NARROW>::WARPS * 32, 1) kv_chunk_kernel(const ChunkArgs c) {
  constexpr int D = HD, COLS = NARROW ? 32 : KEYS, SETS = NARROW ? 2 : 1;
  using L = LayX;
  using R = Roles<NARROW>;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  const ChunkBars b(reinterpret_cast<uint64_t*>(smem + L::BARS));
  uint64_t *const qfull = b.rest, *const raw = qfull + 2, *const rempty = raw + 8 * SETS;      // raw, rempty: [set][page], of every slot: filled, in registers
  uint32_t* const slot_at = reinterpret_cast<uint32_t*>(smem + L::SLOT);
  const Attn8& a = c.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.Hq / a.H;
  pdl_wait();
  pdl_launch_dependents();
  Work w;
  // (a unit that is not split, among ones that are, leaves a mark for the join: no sum is negative)
  const int splits = (int)blockIdx.x < c.whole ? 1 : c.parts.splits, x = (int)blockIdx.x - c.whole;
  if (!chunk_work<NARROW ? FEW : 2 * ROWS>(a, x < 0 ? blockIdx.x : c.whole + x / splits, x < 0 ? 0 : x % splits, splits, c.slots, G, lane, w)) return;
  const int tiles = max(w.count0, w.count1);
  // (pages behind the last key of the sequence, or behind its row of the table, may not exist: no key of theirs is seen)
  const int end_page = min((w.pos0 + w.n - 1) / PAGE + 1, a.table_width);
  const uint64_t keep = policy_evict_last();                      // other row tiles of the sequence read the same pages

  if (warp == R::MMA) {
    if (lane == 0) *reinterpret_cast<Kept*>(smem + L::KEPT) = {w.row0, w.rows, w.first, w.h, w.split, splits, w.b, w.pos0, w.lo0, {0x7FFFFFFF, -1, {}, {}}};
    if (elect_one()) {
      mbar_init(qfull, 4);
      mbar_init(qfull + 1, 4);
      b.init(TILE_PAGES);
    }
    __syncwarp();
    tmem_alloc<1>(slot_at, 512);
    tmem_relinquish<1>();
  }
  // (the first pages are requested before the roles meet; q, which takes its time, is nobody's but the MMAs' to wait for)
  auto meet = [] {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };

  if (warp < R::CONV) {
    if (R::R_SOFTMAX > R::R_START) regs_up<R::R_SOFTMAX>();
    // ---------------------------------------------------------------- softmax: this thread's row
    const int t = warp >> 2, count = t ? w.count1 : w.count0, my = w.row0 + (NARROW ? lane : t * ROWS + (warp & 3) * 32 + lane);
    const bool live = my < w.row0 + w.rows;
    const int pos = w.pos0 + (live ? my / G : 0);
    // (a row that is none sees everything: its results go nowhere, and a warp with one does not take the masked way for it)
    const int hi = live ? min(pos, a.table_width * PAGE - 1) : 0x7FFFFFFF, lo = !live ? 0 : window_from(a.window, pos, w.lo0);
    const bool any = __any_sync(FULL, live);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    meet();
    // ---- the warp's 32 rows of q: sixteen lanes read a row (rows that are none: the last one again)
    if (count > 0) {
      const int last = w.row0 + w.rows - 1, col = lane & 15;
      int row = my - lane + (lane >> 4);
      RowWalk at(min(row, last), G);
      uint4 u[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        u[i] = *reinterpret_cast<const uint4*>(a.q + (long long)(w.first + at.token) * a.q_stride + (w.h * G + at.head) * D + 8 * col);
        row += 2;
        at.step(row <= last ? 2 : 0);
      }
      uint8_t* const rows = smem + L::Q + t * L::TILE + (warp & 3) * (32 * 128) + (col >> 3) * L::HALF;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 2 * i + (lane >> 4);
        *reinterpret_cast<uint4*>(rows + r * 128 + (((col & 7) ^ (r & 7)) << 4)) = u[i];
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(qfull + t);
    }
    const uint32_t tmem = *slot_at + ((uint32_t)((warp & 3) * 32) << 16), ts = tmem + t * 128, to = tmem + 256 + t * D;
    // The second row tile begins when the first has its first P: from then on each has the special function units to itself while the
    // other's products run.  (A barrier of its own, which completes once: the first tile's softmax does not wait for this one's, so that
    // it could complete a phase of `pfull` and the next before a warp here has looked)
    if (t == 1 && count > 0 && w.count0 > 0) ok = mbar_wait(b.begin1, 0);
    for (int j = 0; ok && j < count; ++j) {
      if (!mbar_wait_look(b.sfull + t, (uint32_t)j & 1u)) { ok = false; break; }
      tc_fence_after();
      if (any) {
        // (NARROW: this warp's own 32 of the columns)
        const int k0 = (w.first_tile + j) * KEYS + (NARROW ? 32 * warp : 0), l0 = lo - k0, l1 = hi - k0;       // this row sees columns l0 .. l1
        // ---- the row's scores, all of them in registers; what it does not see is -inf
        uint32_t v[COLS];
#pragma unroll
        for (int q = 0; q < COLS / 32; ++q) tm_ld32(ts + 32 * q + (NARROW ? 32 * warp : 0), v + 32 * q);
        tm_wait_ld<COLS>(v);
        if (__any_sync(FULL, l0 > 0 || l1 < COLS - 1)) {
#pragma unroll
          for (int k = 0; k < COLS; ++k) v[k] = k < l0 || k > l1 ? 0xFF800000u : v[k];
        }
        float x = __uint_as_float(v[0]), y = __uint_as_float(v[1]);
#pragma unroll
        for (int k = 2; k < COLS - 2; k += 4) {
          x = max3(x, __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
          y = max3(y, __uint_as_float(v[k + 2]), __uint_as_float(v[k + 3]));
        }
        x = max3(x, __uint_as_float(v[COLS - 2]), __uint_as_float(v[COLS - 1]));
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
        for (int q = 0; q < COLS / 32; ++q) {
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
          tm_st16(ts + 16 * q + (NARROW ? 16 * warp : 0), pk);
          if (!NARROW && q == 1) {                                           // the product with the first 64 keys need not wait for the others
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b.pfull + t);
          }
        }
        if (NARROW) {                                             // the other columns are other warps' (their copy of the row)
          const uint32_t none[16] = {};
#pragma unroll
          for (int q = 1; q < 4; ++q) tm_st16(ts + 16 * ((warp + q) & 3), none);
        }
        float s0, s1;
        unpair2(sum, s0, s1);
        l += s0 + s1;
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (NARROW || !any) mbar_arrive(b.pfull + t);
        mbar_arrive(b.pfull + 2 + t);
        if (t == 0 && j == 0) mbar_arrive(b.begin1);
      }
    }
    if (ok && count > 0) ok = mbar_wait(b.ofull + t, 0);
    if (!ok && lane == 0) atomicExch(c.status, ERR_WAIT_ACC);
    // ---- out (a wait that ran out leaves the rows unwritten).  Where the rows go comes back from shared memory: held across the loop it cost
    // registers there (2048 queries behind 30000 tokens 1180 us, so 1117)
    const Kept& kept = *reinterpret_cast<const Kept*>(smem + L::KEPT);
    Work o;
    Parts8 parts = c.parts;
    o.row0 = kept.row0; o.rows = kept.rows; o.first = kept.first; o.h = kept.h; o.split = kept.split;
    parts.splits = kept.splits;
    const int row = o.row0 + (NARROW ? lane : t * ROWS + (warp & 3) * 32 + lane), of = a.Hq / a.H;
    const bool mine = row < o.row0 + o.rows;
    const int token = mine ? row / of : 0, hq = o.h * of + (mine ? row % of : 0);
    if (kept.splits < c.parts.splits && mine && (!NARROW || warp == 0))
      c.parts.ml[((long long)(o.first + token) * a.Hq + hq) * c.parts.splits * 2 + 1] = -1.f;
    auto leave = [&](const auto last) {
      if (NARROW) {
        narrow_store(a, parts, o, smem, warp, lane, ok, count, to, m, l, last);
      } else if (ok && any) {
        chunk_store<D, true>(a, parts, o, smem, t, warp, lane, mine, token, hq, count, to, m, l, last);
      }
    };
    // (what the rows here see was noted before the arrivals that their products waited for; converters of the other row tile's later keys may
    // still be at it, so that one lane reads for all.  The rare way out apart from the usual one: in its loops a prompt of 4096 took 4 us more)
    const int page1 = __shfl_sync(FULL, *const_cast<const volatile int*>(&kept.beyond.page1), 0);
    if (__builtin_expect(page1 < 0, 1)) {
      leave(AsTheyAre());
    } else {
      const int page0 = __shfl_sync(FULL, *const_cast<const volatile int*>(&kept.beyond.page0), 0);
      leave([&](int q) {
        const int at = kept.pos0 + token, last_key = mine ? min(at, a.table_width * PAGE - 1) : -1;
        return beyond_seen(a, c.pool, kept, page0, page1, q, window_from(a.window, at, kept.start), last_key, NARROW ? warp : -1, lane);
      });
    }
    tc_fence_before();
  } else if (warp < R::MMA) {
    if (R::R_CONV < R::R_START) regs_down<R::R_CONV>();
    // ---------------------------------------------------------------- converters: records -> operand tiles
    const int cw = (warp - R::CONV) % TILE_PAGES, only = (warp - R::CONV) / TILE_PAGES;
    meet();
    bool ok = true;
    for (int j = 0; ok && j < tiles; ++j) {
      const int s = j & 1;
#pragma unroll 1                                                  // (twice the code costs more, in instruction fetches, than it saves)
      for (int kvi = NARROW ? only : 0; kvi < (NARROW ? only + 1 : 2); ++kvi) {
        const int n = 2 * j + kvi, set = n % SETS;                // the n-th fetch of this page's
        ok = mbar_wait_look(raw + 8 * set + cw, (uint32_t)(n / SETS) & 1u);
        if (!ok) break;
        const int first = (w.first_tile + j) * KEYS + cw * PAGE;                  // position of the page's first token
        const bool edge = kvi && (first < w.start || first + PAGE > w.len);
        uint32_t A[2][4][4];
        Lists l;
        bool beyond = false;
        if (first < end_page * PAGE) {
          RecRegs r[2];
          page_take(smem + L::slot(set, cw), lane, r, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(rempty + 8 * set + cw);
          page_lists<NARROW>(l, r, c.pool, kvi, lane);
          beyond = l.beyond;
          decode_frag(r[0], A[0]);
          decode_frag(r[1], A[1]);
          if (edge) page_edge(A, first, w.start, w.len, lane);
        } else {                                                // (a page that is not there: zeros)
          if (lane == 0) mbar_arrive(rempty + 8 * set + cw);
          l.heads = 0u;
#pragma unroll
          for (int i = 0; i < 32; ++i) A[i >> 4][(i >> 2) & 3][i & 3] = 0u;
        }
        // K's stage is free when the scores of tile j - 2 are, V's when its products are: see the commits of the MMA loop
        const int e = kvi ? j - 1 : j - 2;
        if (j > 1) ok = mbar_wait_look(b.empty + (e & 1), (uint32_t)(e >> 1) & 1u);
        if (!ok) break;
        uint8_t* const tile = smem + (kvi ? L::V : L::K) + s * L::TILE + cw * (PAGE * 128);
        page_store<L::HALF>(tile, A, lane);
        page_patch<L::HALF>(tile, l, c.pool, edge, first, w.start, w.len, lane);
        if (beyond) page_finite<L::HALF>(tile, first / PAGE, &reinterpret_cast<Kept*>(smem + L::KEPT)->beyond, lane);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive((kvi ? b.vfull : b.kfull) + s);
      }
    }
    if (!ok && lane == 0) atomicExch(c.status, ERR_WAIT_EMPTY);
  } else {
    regs_down<R::R_MMA>();
    if (warp == R::MMA) {
      // -------------------------------------------------------------- MMAs.  V is read as it lies (dims contiguous: MN-major)
      meet();
      if (elect_one())
        issue_mmas<D, mma_idesc(128, KEYS), mma_idesc(128, D) | 1u << 16>(smem, b, *slot_at, tiles, w.count0, w.count1, c.status, qfull);
      __syncwarp();
      tc_fence_before();
    } else {
      // -------------------------------------------------------------- producers: pages -> slots, a key tile's keys, then its values; warp f
      // brings pages f, f + 3, f + 6 of the eight
      const int f = warp - R::FETCH, FETCHERS = R::FETCHERS;
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
      if (lane < 8 * SETS && lane % 8 % FETCHERS == f) {
        mbar_init(raw + lane, 1);
        mbar_init(rempty + lane, 1);
        fence_barrier_init();
      }
      __syncwarp();
      int now = entry(0), next = -1;
      auto fetch = [&](int i, int n, int e) {                     // keys (n even) or values of page i of a tile
        if (elect_one()) {
          uint64_t* const bar = raw + 8 * (n % SETS) + i;
          mbar_expect_tx(bar, e >= 0 ? (uint32_t)L::SLOT_BYTES : 0u);
          if (e >= 0) bulk_g2s(smem + L::slot(n % SETS, i), head_pages + e * page_step + (n & 1) * L::SLOT_BYTES, L::SLOT_BYTES, bar, keep);
        }
        __syncwarp();
      };
      if (tiles > 0)
        for (int n = 0; n < SETS; ++n)
          for (int i = f; i < 8; i += FETCHERS) fetch(i, n, __shfl_sync(FULL, now, i));
      meet();
      bool ok = true;
      for (int j = 0; ok && j < tiles; ++j) {
        if ((j & 3) == 0) next = entry(j + 4);
#pragma unroll 1
        for (int n = max(2 * j, SETS); ok && n < 2 * j + 2; ++n) {
          int i = f;
          for (; i < 8; i += FETCHERS) {
            ok = mbar_wait_look(rempty + 8 * (n % SETS) + i, (uint32_t)(n / SETS - 1) & 1u);
            if (!ok) break;
            fetch(i, n, __shfl_sync(FULL, now, 8 * (j & 3) + i));
          }
          if (!ok) {                                              // copies in flight land before the CTA ends: the last into every slot
            if (lane == 0) atomicExch(c.status, ERR_WAIT_EMPTY);
            for (int k = f; k < 8; k += FETCHERS)
              for (int last = k < i ? n : n - 1, s = 0; s < SETS && last >= s; ++s)
                (void)mbar_wait(raw + 8 * ((last - s) % SETS) + k, (uint32_t)((last - s) / SETS) & 1u);
          }
        }
        if ((j & 3) == 3) now = next;
      }
    }
  }
  __syncthreads();
  if (warp == R::MMA) {
    tc_fence_after();
    tmem_dealloc<1>(*slot_at, 512);
  }
}

template <typename Kernel>
int opt_in(Kernel* kernel, int bytes, int regs, std::atomic<uint64_t>& set) {
  int dev = 0;                                                    // (set: devices whose limit has been raised)
  if (int e = st::cuda_fail(cudaGetDevice(&dev), "st_kv_chunk_attn: device")) return e;
  if (dev <= 63 && (set.load() >> dev & 1)) return 0;
  if (int e = st::cuda_fail(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "st_kv_chunk_attn: shared memory attribute"))
    return e;
  cudaFuncAttributes has;                                         // (with fewer registers a warpgroup would wait for its share for good)
  if (int e = st::cuda_fail(cudaFuncGetAttributes(&has, kernel), "st_kv_chunk_attn: attributes")) return e;
  ST_REQUIRE(has.numRegs == regs, "st_kv_chunk_attn: compiled to %d registers, not %d", has.numRegs, regs);
  if (dev <= 63) set.fetch_or(1ull << dev);
  return 0;
}
template <bool NARROW>
int chunk_launch(ChunkArgs& c, long long units, cudaStream_t st_) {
  static std::atomic<uint64_t> set{0};
  c.slots = (int)(units / c.a.H);
  const long long whole = c.whole < units ? c.whole : units, ctas = whole + (units - whole) * c.parts.splits;
  ST_REQUIRE(ctas < (1ll << 31), "st_kv_chunk_attn: grid too large");
  c.whole = (int)whole;
  if (int e = opt_in(kv_chunk_kernel<NARROW>, LayX::BYTES, Roles<NARROW>::R_START, set)) return e;
  return st::launch("st_kv_chunk_attn launch", kv_chunk_kernel<NARROW>, dim3((unsigned)ctas), dim3(Roles<NARROW>::WARPS * 32), (size_t)LayX::BYTES, st_, c);
}
}  // namespace

extern "C" int64_t st_kv_chunk_attn_workspace_bytes(int64_t T, int64_t Hq, int64_t S) {
  return T <= 0 || Hq <= 0 || S <= 1 ? 0 : T * Hq * S * (st::HD + 2) * 4;
}

extern "C" int st_kv_chunk_attn(const void* q, int64_t qs, int64_t T, int64_t Hq, const int32_t* cu, int64_t B, const void* kv, int64_t nblocks,
                                int64_t Hkv, const uint32_t* pool, int64_t P, const int32_t* bt, int64_t btw, int64_t bts,
                                const int32_t* lens, const int32_t* starts, int64_t window, void* out, int64_t os, float* wo, float* wml,
                                double scale, int64_t S, int64_t whole, void* stream) {
  const char* who = "st_kv_chunk_attn";
  ChunkArgs c;
  if (int e = st::attn8_args(c.a, who, q, qs, T, Hq, cu, B, kv, (const int8_t*)kv, nblocks, Hkv, HD, bt, btw, bts, lens, starts, window, out, os,
                             scale))
    return e;
  ST_REQUIRE(S >= 1 && S <= 1024 && whole >= 0, "%s: splits must be in [1, 1024], unsplit units not negative", who);
  if (T == 0 || B == 0) return 0;
  ST_REQUIRE(pool && P >= 0 && P < (1ll << 31), "%s: null pointer (pool)", who);
  ST_REQUIRE(S == 1 || (wo && wml && st::aligned16(wo)), "%s: split workspace (wo, wml) missing or unaligned", who);
  ST_REQUIRE(cu || T == B, "%s: without cu every sequence has one query", who);
  ST_REQUIRE(nblocks < (1ll << 31), "%s: too many pages", who);
  c.a.scale_log2 = fmaxf(c.a.scale_log2, FLT_MIN);                // (it multiplies the -inf of what a row does not see)
  c.parts = {wo, wml, (int)S, 1};
  c.pool = {pool, (int)P};
  c.whole = S == 1 ? 0 : (int)(whole < (1ll << 30) ? whole : 1ll << 30);
  c.status = st::status_ptr();
  ST_REQUIRE(c.status != nullptr, "%s: no device status word", who);
  const long long G = Hq / Hkv;
  ST_REQUIRE(T * G < (1ll << 31), "%s: too large", who);
  const cudaStream_t st_ = (cudaStream_t)stream;
  auto units_of = [&](long long rows) { return (T * G / rows + B) * Hkv; };                   // (every sequence may leave a tile unfilled)
  ST_REQUIRE(units_of(FEW) < (1ll << 31), "%s: grid too large", who);
  const int e = T * G <= FEW * B ? chunk_launch<true>(c, units_of(FEW), st_) : chunk_launch<false>(c, units_of(2 * ROWS), st_);
  if (e || S == 1) return e;
  return st::merge8("st_kv_chunk_attn merge launch", c.a, c.parts, HD, st_);
}
