// Rows sorted by expert: the table of each expert's rows and scale blocks, and
// the 128x4-blocked address of a row's MXFP4 scales.
//
// offsets[E + 1] (device memory) gives expert e the rows offsets[e] ..
// offsets[e + 1] - 1.  Codes are stored row after row without gaps; the
// scales, whose 128-row blocks cannot be cut, begin a new block with every
// expert: expert e's block 0 is block sum over e' < e of ceil(count / 128).
#pragma once

#include <stdint.h>

namespace nvfp4 {

constexpr int kMaxExperts = 1024;

// Fills row[0 .. E] and blk[0 .. E] (shared memory) with one warp.  Values of
// `offsets` outside [0, rows], or that fall from one expert to the next, are
// clamped (the range is then empty), so no later address leaves the buffers.
__device__ __forceinline__ void load_expert_table(const int* __restrict__ offsets, int E, int rows, int* row, int* blk) {
  const int lane = threadIdx.x & 31;
  constexpr int kBatch = 8;  // loads in flight per lane: 256 experts per round trip
  int row_carry = min(max(offsets[0], 0), rows), blk_carry = 0;
  if (lane == 0) {
    row[0] = row_carry;
    blk[0] = 0;
  }
  for (int base = 0; base < E; base += 32 * kBatch) {
    int v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int e = base + 32 * i + lane;
      v[i] = e < E ? min(max(offsets[e + 1], 0), rows) : 0;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (base + 32 * i >= E) break;
      int hi = max(v[i], row_carry);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, hi, d);
        if (lane >= d) hi = max(hi, o);
      }
      int lo = __shfl_up_sync(0xffffffffu, hi, 1);
      if (lane == 0) lo = row_carry;
      int nb = (hi - lo + 127) >> 7;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, nb, d);
        if (lane >= d) nb += o;
      }
      nb += blk_carry;
      const int e = base + 32 * i + lane;
      if (e < E) {
        row[e + 1] = hi;
        blk[e + 1] = nb;
      }
      row_carry = __shfl_sync(0xffffffffu, hi, 31);
      blk_carry = __shfl_sync(0xffffffffu, nb, 31);
    }
  }
}

// The expert whose rows hold row r: the number of e with row[e + 1] <= r (E: none).
__device__ __forceinline__ int expert_of(const int* row, int E, int r) {
  int lo = 0, hi = E;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (row[mid + 1] <= r)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// Byte offset of the 4 scales of K columns [128 j, 128 j + 128) of scale row s,
// K128 blocks per 128 rows.
__device__ __forceinline__ int64_t mx_scale_word(int64_t s, int j, int K128) {
  return ((s >> 7) * K128 + j) * 512 + (s & 31) * 16 + ((s & 127) >> 5) * 4;
}

}  // namespace nvfp4
