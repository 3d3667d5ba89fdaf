// The lossless KV page to its readers (st_kv.cu: decode attention; st_kv_chunk.cu: attention of chunks).  A page of one KV head is 6400 bytes:
// keys, then values, each two units of 1600 bytes (dims 0 .. 63 and 64 .. 127), each a record of 16 tokens and its escapes.
#pragma once
#include "st_common.cuh"

namespace st {
constexpr int PAGE_BYTES = 4 * RKV;

// exact bits of one element of a decoded record; the entry is the same in every lane, so the register it lands in is
// warp-uniform and only the lane that owns the element takes the (single) branch
__device__ __forceinline__ void put_exact(uint32_t (&R)[4][4], uint32_t entry, int lane) {
  const int row = (int)((entry >> 6) & 15u), col = (int)(entry & 63u);
  if (lane != (row & 7) * 4 + ((col & 7) >> 1)) return;
  const uint32_t sh = 16u * (uint32_t)(col & 1), keep = ~(0xFFFFu << sh), val = (entry >> 16) << sh;
  switch ((col >> 4) * 4 + (row >> 3) + 2 * ((col >> 3) & 1)) {
#define ST_PUT(i) case i: R[(i) >> 2][(i) & 3] = (R[(i) >> 2][(i) & 3] & keep) | val; break;
    ST_PUT(0) ST_PUT(1) ST_PUT(2) ST_PUT(3) ST_PUT(4) ST_PUT(5) ST_PUT(6) ST_PUT(7)
    ST_PUT(8) ST_PUT(9) ST_PUT(10) ST_PUT(11) ST_PUT(12) ST_PUT(13) ST_PUT(14) ST_PUT(15)
#undef ST_PUT
  }
}

// `n` entries that lanes from, from + 1, ... hold, in their order, put into a unit's decoded fragments
__device__ __forceinline__ void put_list(uint32_t (&R)[4][4], uint32_t entry, int from, int n, int lane) {
  for (int i = 0; i < n; ++i) put_exact(R, __shfl_sync(FULL, entry, from + i), lane);
}
// the escapes of a unit whose slots lie in `entry` from lane `from` on, its first pool block in `word`
__device__ __forceinline__ void unit_escapes(uint32_t head, uint32_t entry, uint32_t word, int from, const uint32_t* pool, int pool_blocks,
                                             int lane, uint32_t (&R)[4][4]) {
  put_list(R, entry, from, min((int)(head & 15u), NSLOT), lane);
  if (!(head & 16u)) return;
  int blk = (int)(head >> 8);
  for (int hops = 0; blk >= 0 && blk < pool_blocks && hops < 4096; ++hops) {
    if (hops > 0) word = __ldg(pool + (size_t)blk * 16 + (lane & 15));
    const uint32_t w0 = __shfl_sync(FULL, word, from);
    put_list(R, word, from + 1, min((int)(w0 & 0xFFu), XSLOT), lane);
    blk = (int)(w0 >> 8) - 1;
  }
}
// the two units (dims 0..63, 64..127) of a page's keys or values in shared memory -> the lane's fragment registers.  Both
// are decoded before the first escape is looked at: two independent chains instead of one.  Half a warp fetches each unit's slots and, where
// there is one, the first block of its chain, ahead of the decoding (an entry at a time, a chain cost a trip to L2 per entry)
__device__ __forceinline__ void units_to_frag(const uint8_t* unit, const uint32_t* pool, int pool_blocks, int lane,
                                              uint32_t (&R)[2][4][4]) {
  const uint32_t h0 = *reinterpret_cast<const uint32_t*>(unit + REC), h1 = *reinterpret_cast<const uint32_t*>(unit + RKV + REC);
  const RecRegs r0 = load_rec_shared(unit, lane), r1 = load_rec_shared(unit + RKV, lane);
  uint32_t entry = 0u, word = 0u;
  if (((h0 | h1) & 31u) != 0u) {
    const uint32_t mine = lane < 16 ? h0 : h1;
    entry = *reinterpret_cast<const uint32_t*>(unit + (lane >> 4) * RKV + REC + 4 + 4 * min(lane & 15, NSLOT - 1));
    if ((mine & 16u) && (int)(mine >> 8) < pool_blocks) word = __ldg(pool + (size_t)(mine >> 8) * 16 + (lane & 15));
  }
  decode_frag(r0, R[0]);
  decode_frag(r1, R[1]);
  if (((h0 | h1) & 31u) == 0u) return;
  unit_escapes(h0, entry, word, 0, pool, pool_blocks, lane, R[0]);
  unit_escapes(h1, entry, word, 16, pool, pool_blocks, lane, R[1]);
}

__device__ __forceinline__ float max_over_rows(float v) {        // lanes that differ in g (bits 2..4) hold other tokens
  v = fmaxf(v, __shfl_xor_sync(FULL, v, 4));
  v = fmaxf(v, __shfl_xor_sync(FULL, v, 8));
  return fmaxf(v, __shfl_xor_sync(FULL, v, 16));
}
__device__ __forceinline__ float sum_over_rows(float v) {
  v += __shfl_xor_sync(FULL, v, 4);
  v += __shfl_xor_sync(FULL, v, 8);
  return v + __shfl_xor_sync(FULL, v, 16);
}
}  // namespace st
