// What the two chunk attentions on the tensor cores share (st_kv8_chunk.cu: pages in 8 bits, st_kv_chunk.cu: lossless pages): the division of
// the rows, shared- and tensor-memory operands, the loop that issues the MMAs, and the way out of a CTA's rows.
#pragma once
#include <type_traits>

#include "st_kv8.cuh"
#include "st_tc.cuh"

namespace st {
constexpr int KEYS = 128, TILE_PAGES = KEYS / PAGE, ROWS = 128;
constexpr int W_CONV = 8;                                         // softmax warps 0 .. 7 (tile = warp / 4), converter warps from here

// Shared memory: the operand tiles, 64 values of a row in 128 bytes with the 128-byte swizzle
template <int D>
struct Tiles {
  static constexpr int HALF = 128 * 128;                          // 128 rows x 64 values of two bytes
  static constexpr int TILE = D / 64 * HALF;
  static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, END = 6 * TILE;      // two tiles of Q, two stages of K and V
};

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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               :: "r"(addr), ST_I4(v, 0), ST_I4(v, 4), ST_I4(v, 8), ST_I4(v, 12) : "memory");
}
#undef ST_R4
#undef ST_I4
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }

// the first key that position `pos` sees (window 0: from start on); pos may be negative (a sequence shorter than its queries)
__device__ __forceinline__ int window_from(int window, int pos, int start) {
  return window > 0 ? (int)max((long long)start, (long long)pos - window + 1) : start;
}
// What a CTA works on; the same in all of its threads
struct Work : Rows8 {
  int h, split, pos0;                                             // position of query 0
  int lo0, first_tile, tiles, count0, count1;                     // key tiles of the split; of those, how many each row tile needs
};
// part `split` of `splits` of unit x (a tile of TILE rows and a KV head).  false: there are no such rows.  Later tiles of a sequence see more
// keys: they go first
template <int TILE>
__device__ __forceinline__ bool chunk_work(const Attn8& a, int x, int split, int splits, int slots, int G, int lane, Work& w) {
  w.split = split;
  w.h = x % a.H;
  if (!find_rows<TILE>(a, G, slots - 1 - x / a.H, lane, w)) return false;
  const int start = w.start;
  w.pos0 = w.len - w.n;
  const int first_pos = w.pos0 + w.row0 / G, last_pos = w.pos0 + (w.row0 + w.rows - 1) / G;
  w.lo0 = start;
  const int lo = window_from(a.window, first_pos, start);
  const int end = (int)min((long long)last_pos + 1, (long long)a.table_width * PAGE);            // keys [lo, end)
  const int t0 = lo / KEYS, t1 = end > lo ? (end - 1) / KEYS + 1 : t0;
  const int per = (t1 - t0 + splits - 1) / splits;
  w.first_tile = t0 + w.split * per;
  w.tiles = max(0, min(t1, w.first_tile + per) - w.first_tile);
  const int mid_pos = w.pos0 + (w.row0 + min(w.rows, ROWS) - 1) / G;                   // last position of the first row tile
  w.count0 = mid_pos < 0 ? 0 : max(0, min(w.tiles, mid_pos / KEYS + 1 - w.first_tile));
  w.count1 = w.rows > ROWS ? w.tiles : 0;
  return true;
}

// The barriers of the hand-overs (pfull: [half of the keys][row tile]; begin1: the second row tile may begin; drain: the way out of an
// issuer that gave up)
struct ChunkBars {
  uint64_t *begin1, *kfull, *vfull, *sfull, *pfull, *ofull, *empty, *drain, *rest;
  static constexpr int COUNT = 17;
  __device__ explicit ChunkBars(uint64_t* b)
      : begin1(b), kfull(b + 2), vfull(b + 4), sfull(b + 6), pfull(b + 8), ofull(b + 12), empty(b + 14), drain(b + 16), rest(b + 17) {}
  __device__ void init(int converters) const {                    // one thread; an arrival per converter warp, or per softmax warp of a row tile
    for (int i = 0; i < 2; ++i) {
      mbar_init(kfull + i, converters);
      mbar_init(vfull + i, converters);
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
};

// The MMAs of a CTA's two row tiles (of `count0` and `count1` key tiles).  One thread's MMAs complete in the order of their issue (and a
// commit covers all before it): S of the next key tile may take the place of the P that the product before it reads.
// The whole loop runs in one elected thread, waits included: a warp that meets again around each step costs more than the steps.
// qfull: a barrier per row tile that says its q is in shared memory (nullptr: it is)
template <int D, uint32_t IDESC_S, uint32_t IDESC_O>
__device__ __forceinline__ void issue_mmas(uint8_t* const smem, const ChunkBars& b, uint32_t tmem, int tiles, int count0, int count1, int* status,
                                           uint64_t* qfull = nullptr) {
  const uint32_t dq = desc_k(smem_addr(smem + Tiles<D>::Q)), dk = desc_k(smem_addr(smem + Tiles<D>::K)), dv = desc_mn(smem_addr(smem + Tiles<D>::V), Tiles<D>::HALF);
  auto scores = [&](int t, int s) {
    const uint32_t q = dq + t * (Tiles<D>::TILE >> 4), k = dk + s * (Tiles<D>::TILE >> 4);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint32_t at = (i >> 2) * (Tiles<D>::HALF >> 4) + 2 * (i & 3);
      mma_ss(tmem + t * 128, q + at, k + at, IDESC_S, i > 0);
    }
    tc_commit(b.sfull + t);
  };
  auto outputs = [&](int t, int s, int half, bool more) {
    const uint32_t v = dv + s * (Tiles<D>::TILE >> 4);
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
    ok = mbar_wait(b.kfull, 0);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (ok && (t ? count1 : count0) > 0 && (!qfull || (ok = mbar_wait(qfull + t, 0)))) {
        tc_fence_after();
        scores(t, 0);
      }
  }
  for (int j = 0; ok && j < tiles; ++j) {
    const int s = j & 1, s1 = s ^ 1;
    ok = mbar_wait_look(b.vfull + s, (uint32_t)(j >> 1) & 1u);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int count = t ? count1 : count0;
      if (!ok || j >= count) continue;
      ok = mbar_wait_look(b.pfull + t, (uint32_t)j & 1u);
      if (!ok) continue;
      tc_fence_after();
      outputs(t, s, 0, j > 0);
      ok = mbar_wait_look(b.pfull + 2 + t, (uint32_t)j & 1u);
      if (!ok) continue;
      tc_fence_after();
      outputs(t, s, 1, true);
      if (t == 0 || j >= count0) tc_commit(b.empty + s);
      if (j + 1 < count) {
        ok = mbar_wait_look(b.kfull + s1, (uint32_t)((j + 1) >> 1) & 1u);
        if (!ok) continue;
        tc_fence_after();
        scores(t, s1);
      } else {
        tc_commit(b.ofull + t);
      }
    }
  }
  if (!ok) {                                                  // (gave up: let what was issued complete before the memory goes)
    atomicExch(status, ERR_WAIT_MMA);
    tc_commit(b.drain);
    (void)mbar_wait(b.drain, 0);
  }
}
// Walks rows (query, head of the group) of a sequence in steps, without a division a step; and without a shuffle: shuffles between loads wait
// for them (sixteen rows of q took 7000 cycles to ask for, one after the other)
struct RowWalk {
  int token, head, G;
  __device__ RowWalk(int row, int group) : token(row / group), head(row % group), G(group) {}
  __device__ __forceinline__ void step(int rows) {
    head += rows;
    while (head >= G) { head -= G; ++token; }
  }
};
// A softmax warp's rows leave: this lane's row of O (tensor memory `to`, key tiles seen: count) over its sum l, or, of a split, as it is
// with (reference m, l).  The whole warp calls.  last(q).to(v) has the last word on values 32 q .. 32 q + 31 of the lane's row
struct AsTheyAre {
  __device__ __forceinline__ AsTheyAre operator()(int) const { return {}; }
  __device__ __forceinline__ void to(uint32_t*) const {}
};
// WALK: where the rows lie is walked to, from w, by code that is not unrolled; else it comes from the lanes that own them (live, token, hq).  Of two
// ways to the same end each kernel has the one whose registers leave its loop alone: 8-bit pages 2048 queries behind 30000 tokens 1024 us walked,
// 960 not, nine chunks of dimension 64 52.9 and 52.1; lossless pages, with w from shared memory, a prompt of 4096 179 and 184
template <int D, bool WALK, class Last = AsTheyAre>
__device__ __forceinline__ void chunk_store(const Attn8& a, const Parts8& parts, const Work& w, uint8_t* const smem, int t, int warp, int lane,
                                            bool live, int token, int hq, int count, uint32_t to, float m, float l, const Last last = Last()) {
  tc_fence_after();
  const long long r = (long long)(w.first + token) * a.Hq + hq;
  const float inv = parts.splits > 1 ? 1.f : (l > 0.f ? 1.f / l : l);
  if (live && parts.splits > 1) {
    float* const ml = parts.ml + (r * parts.splits + w.split) * 2;
    ml[0] = l > 0.f || l != l ? m : -INFINITY;
    ml[1] = l;
  }
  if (parts.splits > 1) {
    float* const o = parts.o + (r * parts.splits + w.split) * D;
    constexpr int AT_ONCE = std::is_same_v<Last, AsTheyAre> ? D / 32 : 1;
#pragma unroll AT_ONCE
    for (int q = 0; q < D / 32; ++q) {
      const auto more = last(q);                                  // (while no values are held)
      uint32_t v[32];
      if (count > 0) {
        tm_ld32(to + 32 * q, v);
        tm_wait_ld<32>(v);
      }
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = count > 0 && l != 0.f ? __float_as_uint(__uint_as_float(v[k]) * inv) : 0u;
      more.to(v);
      if (live)
#pragma unroll
        for (int k = 0; k < 8; ++k) reinterpret_cast<uint4*>(o + 32 * q)[k] = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      __syncwarp();
    }
  } else {
    // the warp's rows leave through where its rows of q were (their last scores are done), D / 8 lanes a row
    constexpr int LANES = D / 8, PER = 32 / LANES;
    uint8_t* const rows = smem + Tiles<D>::Q + t * Tiles<D>::TILE + (warp & 3) * (32 * 2 * D);
    constexpr int AT_ONCE = WALK ? 1 : D / 32;                    // (code that runs once: what it costs is to be fetched)
#pragma unroll AT_ONCE
    for (int q = 0; q < D / 32; ++q) {
      const auto more = last(q);                                  // (while no values are held)
      uint32_t v[32];
      if (count > 0) {
        tm_ld32(to + 32 * q, v);
        tm_wait_ld<32>(v);
      }
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = count > 0 && l != 0.f ? __float_as_uint(__uint_as_float(v[k]) * inv) : 0u;
      more.to(v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = pack_bf16(__uint_as_float(v[8 * k + 2 * i]), __uint_as_float(v[8 * k + 2 * i + 1]));
        *reinterpret_cast<uint4*>(rows + lane * (2 * D) + (((4 * q + k) ^ (lane & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
    __syncwarp();
    if constexpr (WALK) {
      int row = lane / LANES;
      const int at = t * ROWS + (warp & 3) * 32 + row, G = a.Hq / a.H;
      RowWalk to_row(w.row0 + at, G);
#pragma unroll 4
      for (int i = 0; i < LANES; ++i, row += PER, to_row.step(PER))
        if (at + i * PER < w.rows)
          *reinterpret_cast<uint4*>(a.out + (long long)(w.first + to_row.token) * a.out_stride + (w.h * G + to_row.head) * D + 8 * (lane % LANES)) =
              *reinterpret_cast<const uint4*>(rows + row * (2 * D) + (((lane % LANES) ^ (row & 7)) << 4));
    } else {
      const long long mine = live ? (long long)(w.first + token) * a.out_stride + (long long)hq * D : -1;
#pragma unroll
      for (int i = 0; i < LANES; ++i) {
        const int row = i * PER + lane / LANES;
        const long long to_row = __shfl_sync(FULL, mine, row);
        if (to_row >= 0)
          *reinterpret_cast<uint4*>(a.out + to_row + 8 * (lane % LANES)) =
              *reinterpret_cast<const uint4*>(rows + row * (2 * D) + (((lane % LANES) ^ (row & 7)) << 4));
      }
    }
  }
}
}  // namespace st
