// Shared by the kernels of the ragged expert products: the tiles of a device-side list of groups.
//
// Group e holds the rows [o_e, o_{e+1}) of `offsets`.  The list comes from device memory, so kernels never trust it: an
// entry counts as the largest value seen so far and as n at most, which keeps every row index inside the tensors.
#pragma once

#include <cstdint>

#include "common.cuh"
#include "elem.cuh"

namespace sb {

constexpr int kMaxGroups = 1024;

struct GroupTile {
  int expert;          // -1: the tile does not exist
  int index;           // number of the tile inside its group
  int begin, end;      // rows of the group
};

__device__ __forceinline__ int clamped_offset(const int32_t *offsets, int e, int n) {
  const int v = offsets[e];
  return v < 0 ? 0 : v > n ? n : v;
}

// Pieces of `rows` rows that `length` rows make, and where the piece from row `begin` on ends.  (Row numbers reach 2^31: the
// sum of two of them does not fit their type.)
__device__ __forceinline__ int pieces_of(int length, int rows) {
  return static_cast<int>((static_cast<uint32_t>(length) + static_cast<uint32_t>(rows) - 1u) / static_cast<uint32_t>(rows));
}
__device__ __forceinline__ int piece_end(int begin, int end, int rows) { return end - begin > rows ? begin + rows : end; }

// The t-th tile of `rows` rows over all groups, found by one whole warp (every lane gets the answer).
__device__ __forceinline__ GroupTile find_group_tile(const int32_t *offsets, int experts, int n, int rows, int t) {
  const int lane = threadIdx.x & 31;
  GroupTile r{-1, 0, 0, 0};
  int tiles_before = 0, highest = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int e = e0 + lane;
    int hi = e < experts ? clamped_offset(offsets, e + 1, n) : 0;
    int lo = e < experts ? clamped_offset(offsets, e, n) : 0;
    // running maximum: begin of group e = largest of offsets[0..e]
    int run = lo;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, run, d);
      if (lane >= d && o > run) run = o;
    }
    lo = run > highest ? run : highest;
    hi = hi > lo ? hi : lo;
    if (e >= experts) hi = lo;
    const int mine = pieces_of(hi - lo, rows);
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const int first = tiles_before + sum - mine;
    const uint32_t hit = __ballot_sync(0xffffffffu, t >= first && t < first + mine);
    if (hit != 0) {
      const int src = __ffs(hit) - 1;
      r.expert = e0 + src;
      r.index = t - __shfl_sync(0xffffffffu, first, src);
      r.begin = __shfl_sync(0xffffffffu, lo, src);
      r.end = __shfl_sync(0xffffffffu, hi, src);
      return r;
    }
    tiles_before += __shfl_sync(0xffffffffu, sum, 31);
    highest = __shfl_sync(0xffffffffu, hi > lo ? hi : lo, 31);
  }
  return r;
}

// First and last row of all groups together (the same clamping as above).
__device__ __forceinline__ void group_span(const int32_t *offsets, int experts, int n, int &first, int &last) {
  first = clamped_offset(offsets, 0, n);
  last = first;
  for (int e = 1; e <= experts; ++e) {
    const int v = clamped_offset(offsets, e, n);
    last = v > last ? v : last;
  }
}

// upper bound of the number of tiles of `rows` rows, for a host that does not know the offsets
inline int64_t group_tiles_bound(int64_t n, int experts, int64_t rows) { return n / rows + (experts < n ? experts : n); }

// Bytes per row of the ReLU mask: a bit per column, rows of whole 4-byte words.
__host__ __device__ __forceinline__ int mask_pitch(int c_out) { return (c_out + 31) / 32 * 4; }

inline int pitch8(int channels) { return (channels + 7) / 8 * 8; }

// The tensor-core path (grouped_tc.cu).  Channel counts are free; tensors and rows start on 16-byte boundaries, so weights and
// results have pitches (elements per row) in whole units of 8.
enum { kForward = 0, kDx = 1, kDw = 2 };
bool grouped_tc_available();
bool grouped_tc_pair(int mode, const spira_b200_grouped_desc &D);      // whether pairs of CTAs share its tiles
bool grouped_tc_rows_ok(const void *p, int64_t stride, int channels, int64_t n);
int grouped_tc_dw_tiles(int c_in, int c_out);
int grouped_tc_run(int mode, const spira_b200_grouped_desc &D, int w_pitch, int out_pitch, int piece, float *partial, int32_t *status,
                   unsigned long long wait_ns, cudaStream_t st);

}  // namespace sb
