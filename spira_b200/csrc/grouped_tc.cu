// Ragged products on the fifth-generation tensor cores: tcgen05.mma with operands moved by TMA, accumulators in tensor memory.
//
//   forward   y[rows of e]  = x W[e]       M = rows,  N = c_out, K = c_in    A = x  (K-major),  B = W[e]  (N-major)
//   dx        dx[rows of e] = dz W[e]^T    M = rows,  N = c_in,  K = c_out   A = dz (K-major),  B = W[e]  (K-major)
//   dW        dW[e] = x_e^T dz_e           M = c_in,  N = c_out, K = rows    A = x  (M-major),  B = dz    (N-major)
//
// No operand is transposed or copied: the three products read the same tensors and differ in the majors of the instruction
// descriptor and in the boxes TMA fetches (128-byte swizzle everywhere).  A tile has 128 rows of M; rows past the end of a
// group belong to the next one, they are multiplied and not stored.  In dW the rows are the reduction: the last step of a
// group overwrites foreign rows with zeros in BOTH operands in shared memory (0 * NaN of a neighbour would not be 0).
//
// With many rows per group two CTAs of a cluster share a tile of 256 rows (cta_group::2): each holds its 128 rows of A and
// half of the columns of B, the leader issues the MMAs for both, and every byte of B crosses from L2 to one SM instead of
// two (32 instead of 48 KB per stage, six stages instead of four).
//
// One persistent CTA per SM, 20 warps: warp 0 issues TMA loads, warp 1 the MMAs, warps 4-19 (four per tensor-memory lane
// quarter, a quarter of the columns each) convert and store while the next tile accumulates in the other half of tensor
// memory.  Every CTA reads the group boundaries once into shared memory.  Every wait is bounded; an expired one raises the
// status word.
//
// Measured one at a time behind an L2 flush: 254 726 rows in 8 groups 96 -> 384 fp16 with bias 61 us (a fill of its
// 196 MB of results alone: 53 us); 80 026 rows in 16 groups 512 -> 2048 bf16: forward with bias, ReLU and mask 162 us, dx
// 119 us = 1410 TFLOP/s, dW 136 us (one dense library product of the size on the same board: 139, 115, 126).
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "elem.cuh"
#include "grouped.cuh"
#include "ptx.cuh"

namespace sb {

using namespace sb::ptx;

constexpr int kGRows = 128;                    // M of a tile
constexpr int kGK = 64;                        // reduction per stage: 128 bytes, one swizzle row
constexpr int kGABytes = kGRows * kGK * 2;
constexpr int kGBlock = kGK * 64 * 2;          // one 64 x 64 box
constexpr int kGMaxN = 256;
constexpr int kGMaxStages = 8;
constexpr int kGEpilogueWarps = 16, kGFirstEpilogueWarp = 4;
constexpr int kGThreads = (kGFirstEpilogueWarp + kGEpilogueWarps) * 32;
constexpr int kGSmemBudget = 224 * 1024;
constexpr int kGBiasBytes = kGEpilogueWarps * 64 * 4;   // a warp's columns of the bias as fp32
constexpr int kGSorted = 64;                   // groups up to which dW takes the longest first

struct GroupedTcParams {
  const int32_t *offsets;
  void *out;                 // y, dx or dW
  float *partial;            // dW in pieces: [unit][c_in][c_out]
  const void *bias;
  int32_t *status;
  int n, experts, m_channels, n_channels, k_channels;   // m_channels: c_in in dW; k_channels: 0 in dW (rows)
  int out_pitch;             // elements per row of the result (and of the partial sums): n_channels in whole units of 8 at least
  int relu, piece;           // piece: rows per unit of dW, 0 = whole groups
  int tile_rows;             // M of a tile: 128, or 256 for a pair of CTAs
  int bn, n_tiles, m_tiles;  // columns per tile, column tiles, row tiles of dW
  int stages, b_bytes, acc_stride, tmem_cols, off_bias, off_stage, off_bar, off_groups;
  int box_cols;              // columns of a block that leaves through shared memory and TMA (32 or 48), 0: direct stores
  unsigned char *mask;       // forward: a bit per element that the ReLU let through
  int mask_pitch;
  uint32_t idesc;
  unsigned long long wait_ns;
};

template <bool PAIR>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  if constexpr (PAIR)      // (the barrier may lie in the other CTA of the pair)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// One lane of a converged warp.  MMAs and TMA loads sit behind this and not behind `lane == 0`: the compiler then knows that
// one thread issues and keeps the operands in uniform registers (measured without loads: 93 instead of 146 us for the MMAs
// of 80 026 x 2048 x 512).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// ---- the two CTAs of a pair
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait (kCluster: for arrivals of the other CTA).  The clock is read only after some tries: its latency would be
// added to every step of a loop that finds its barrier not quite ready.
template <bool kCluster>
__device__ __forceinline__ bool group_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, unsigned long long limit_ns) {
  unsigned long long t0 = 0;
  for (int spins = 1; !(kCluster ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)); ++spins) {
    if ((spins & 63) == 0) {
      if (*abort_flag != 0) return false;
      const unsigned long long now = global_timer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > limit_ns) {
        *abort_flag = 1;
        return false;
      }
    }
  }
  return true;
}
// The limit of a wait for something that comes at the end of a tile: it spans all reduction steps of the tile (dW: of a whole
// group, 10^6 rows take 5 ms), so each thousand of them has the limit of one wait to itself.
__device__ __forceinline__ unsigned long long tile_limit(unsigned long long limit_ns, int steps) { return limit_ns * (1 + static_cast<unsigned>(steps) / 1024); }
template <bool PAIR>
__device__ __forceinline__ void group_tmem_alloc(uint32_t dst, uint32_t cols) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, cols);
    tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void group_tmem_dealloc(uint32_t addr, uint32_t cols) {
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  else tmem_dealloc(addr, cols);
}
template <bool PAIR>
__device__ __forceinline__ void group_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    mma_f16_ss(d, a, b, idesc, accumulate);
}
// Arrives once the MMAs issued so far are done: on this CTA's barrier, or on the same barrier of both CTAs.
template <bool PAIR>
__device__ __forceinline__ void group_commit(uint32_t bar) {
  if constexpr (PAIR) {
    const uint16_t both = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(both) : "memory");
  } else {
    mma_commit(bar);
  }
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y),
               "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Operand whose M (or N) elements are contiguous, 128-byte swizzle: 64 x 64 boxes (64 reduction rows of 128 bytes); eight
// reduction rows are 1024 bytes, the next 64 elements of M / N are the next box.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kGBlock >> 4) << 16;      // leading byte offset: next 64 elements of M / N
  d |= static_cast<uint64_t>(1024 >> 4) << 32;         // stride byte offset: next 8 reduction rows
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;                 // 128-byte swizzle
  return d;
}

// Where tile t lies.  Tiles are numbered (group, unit of the group, column tile): neighbouring CTAs share the same rows.
struct TcTile {
  int expert, unit, row0, row_end;     // unit: number of the (group, unit) pair; rows: M of forward / dx, reduction of dW
  int m0, n0;                          // first channel of M (dW) and of N
  int steps;                           // reduction steps of kGK
};

template <int MODE>
struct TileWalk {
  const int *rows, *first, *by_size;   // shared memory: group boundaries, first unit of every group, dW: groups by length
  int place = 0;
  __device__ __forceinline__ TcTile at(const GroupedTcParams &P, int t) {
    TcTile r;
    const int per_unit = MODE == kDw ? P.m_tiles * P.n_tiles : P.n_tiles;
    const int unit = t / per_unit, in_unit = t - unit * per_unit;
    while (unit >= first[place + 1]) ++place;          // (t only grows)
    const int index = unit - first[place];
    const int expert = MODE == kDw && P.piece == 0 && P.experts <= kGSorted ? by_size[place] : place;
    r.expert = expert;
    r.unit = unit;
    r.n0 = in_unit % P.n_tiles * P.bn;
    if (MODE == kDw) {
      r.m0 = in_unit / P.n_tiles * P.tile_rows;
      r.row0 = rows[expert] + index * P.piece;
      r.row_end = P.piece ? piece_end(r.row0, rows[expert + 1], P.piece) : rows[expert + 1];
      r.steps = pieces_of(r.row_end - r.row0, kGK);
    } else {
      r.m0 = 0;
      r.row0 = rows[expert] + index * P.tile_rows;
      r.row_end = rows[expert + 1];
      r.steps = (P.k_channels + kGK - 1) / kGK;
    }
    return r;
  }
};

// Group boundaries (clamped, never falling) and the first unit of every group, by one warp.
template <int MODE>
__device__ __forceinline__ void read_groups(const GroupedTcParams &P, int *rows, int *first, int *by_size) {
  const int lane = threadIdx.x & 31;
  int highest = 0, units = 0;
  for (int e0 = 0; e0 <= P.experts; e0 += 32) {
    const int e = e0 + lane;
    int v = e <= P.experts ? clamped_offset(P.offsets, e, P.n) : 0;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d && o > v) v = o;
    }
    v = v > highest ? v : highest;
    if (e <= P.experts) rows[e] = v;
    highest = __shfl_sync(0xffffffffu, v, 31);
  }
  __syncwarp();
  const int unit_rows = MODE == kDw ? P.piece : P.tile_rows;
  for (int e0 = 0; e0 < P.experts; e0 += 32) {
    const int e = e0 + lane;
    int mine = 0;
    if (e < P.experts) mine = unit_rows == 0 ? 1 : pieces_of(rows[e + 1] - rows[e], unit_rows);
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (e < P.experts) first[e] = units + sum - mine;
    units += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) first[P.experts] = units;
  // whole groups as units of dW: the longest first, so that the last round of CTAs has the short ones
  if (MODE == kDw && P.piece == 0 && P.experts <= kGSorted)
    for (int e = lane; e < P.experts; e += 32) {
      const int mine = rows[e + 1] - rows[e];
      int rank = 0;
      for (int f = 0; f < P.experts; ++f) {
        const int other = rows[f + 1] - rows[f];
        rank += other > mine || (other == mine && f < e);
      }
      by_size[rank] = e;
    }
}

// The tile of worker `me` of G in round r: rounds run over the workers in alternating direction.
__device__ __forceinline__ int round_tile(int r, int me, int G) { return r * G + (r & 1 ? G - 1 - me : me); }

// Two values rounded into one word (a in the low half), negative ones to zero with kRelu (a NaN stays).
template <typename T, bool kRelu>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) {
    if (kRelu) asm("cvt.rn.relu.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  } else {
    if (kRelu) asm("cvt.rn.relu.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  }
  return r;
}

// W (16 or 32) columns of one row of the accumulator: bias, ReLU, one rounding.  `bits` gets a bit per column, set where the
// value is positive (the sign of 0 - v).
template <typename T, int W, bool kRelu>
__device__ __forceinline__ void convert_columns(uint32_t (&r)[W], const float *bias, bool want_bits, uint4 (&v)[W / 8], uint32_t &bits) {
  if (bias) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const float4 b = *reinterpret_cast<const float4 *>(bias + i);
      r[i] = __float_as_uint(__uint_as_float(r[i]) + b.x);
      r[i + 1] = __float_as_uint(__uint_as_float(r[i + 1]) + b.y);
      r[i + 2] = __float_as_uint(__uint_as_float(r[i + 2]) + b.z);
      r[i + 3] = __float_as_uint(__uint_as_float(r[i + 3]) + b.w);
    }
  }
  if (kRelu && want_bits) {
    bits = 0;
#pragma unroll
    for (int i = W - 1; i >= 0; --i) bits = __funnelshift_l(__float_as_uint(0.f - __uint_as_float(r[i])), bits, 1);
  }
#pragma unroll
  for (int h = 0; h < W / 8; ++h) {
    const uint32_t *q = r + 8 * h;
    v[h] = make_uint4(pack2<T, kRelu>(__uint_as_float(q[0]), __uint_as_float(q[1])), pack2<T, kRelu>(__uint_as_float(q[2]), __uint_as_float(q[3])),
                      pack2<T, kRelu>(__uint_as_float(q[4]), __uint_as_float(q[5])), pack2<T, kRelu>(__uint_as_float(q[6]), __uint_as_float(q[7])));
  }
}

// The same row's 16-byte units to global memory, whole 32-byte sectors where they are aligned.
template <typename T, int U>
__device__ __forceinline__ void store_units(const uint4 (&v)[U], T *dst, int valid) {
  const bool wide = (reinterpret_cast<uintptr_t>(dst) & 31) == 0;
#pragma unroll
  for (int h = 0; h < U; h += 2) {
    if (wide && 8 * h + 16 <= valid) {
      st_global_v8(dst + 8 * h, v[h], v[h + 1]);
    } else {
      if (8 * h < valid) *reinterpret_cast<uint4 *>(dst + 8 * h) = v[h];
      if (8 * h + 8 < valid) *reinterpret_cast<uint4 *>(dst + 8 * h + 8) = v[h + 1];
    }
  }
}

// fp32 partial sums of dW: W columns of one row.
template <int W>
__device__ __forceinline__ void store_partial(const uint32_t (&r)[W], float *dst, int valid) {
#pragma unroll
  for (int i = 0; i < W; i += 4)
    if (i < valid) *reinterpret_cast<uint4 *>(dst + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
}

template <typename T, int MODE, bool PAIR>
__global__ void __launch_bounds__(kGThreads, 1) grouped_tc_kernel(const __grid_constant__ GroupedTcParams P, const __grid_constant__ CUtensorMap map_a,
                                                                   const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out) {
  extern __shared__ unsigned char grouped_smem_raw[];
  const uint32_t raw = smem_u32(grouped_smem_raw);
  unsigned char *smem = grouped_smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + P.off_bar;
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (kGMaxStages + s); };
  auto bar_acc_full = [&](int b) { return bar0 + 8u * (2 * kGMaxStages + b); };
  auto bar_acc_empty = [&](int b) { return bar0 + 8u * (2 * kGMaxStages + 2 + b); };
  // dW of a pair, last step of a group: the follower's rows have landed (its own barrier) / are cleaned (the leader's)
  auto bar_tail = [&](int s) { return bar0 + 8u * (2 * kGMaxStages + 4 + s); };
  auto bar_clean = [&](int s) { return bar0 + 8u * (3 * kGMaxStages + 4 + s); };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + P.off_bar + 8 * (4 * kGMaxStages + 4));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + P.off_bar + 8 * (4 * kGMaxStages + 4) + 4);
  int *rows = reinterpret_cast<int *>(smem + P.off_groups), *first = rows + P.experts + 1, *by_size = first + P.experts + 1;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
  const int me = PAIR ? blockIdx.x / 2 : blockIdx.x, G = PAIR ? gridDim.x / 2 : gridDim.x;
  const int stages = P.stages, stage_bytes = kGABytes + P.b_bytes;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
      if (PAIR && MODE == kDw) {
        mbar_init(bar_tail(s), 1);
        mbar_init(bar_clean(s), 1);
      }
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), kGEpilogueWarps * (PAIR ? 2 : 1));
    }
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) group_tmem_alloc<PAIR>(smem_u32(tmem_slot), P.tmem_cols);
  pdl_wait();            // before the first global read of any thread
  if (warp == 2) read_groups<MODE>(P, rows, first, by_size);
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();      // the other CTA's barriers are ready too
  tc_fence_after();
  pdl_trigger();         // (behind the allocation: a CTA of the next kernel on this SM cannot take the tensor memory first)
  const uint32_t tmem_base = *tmem_slot;
  const int total = first[P.experts] * (MODE == kDw ? P.m_tiles * P.n_tiles : P.n_tiles);
  TileWalk<MODE> walk{rows, first, by_size};
  const int rounds = (total + G - 1) / G;
  const int b_columns = PAIR ? P.bn / 2 : P.bn;

  if (warp == 0) {
    // =========================== TMA loads ===========================
    int stage = 0, phase = 0;
    bool ok = true;
    for (int round = 0; ok && round < rounds; ++round) {
      const int t = round_tile(round, me, G);
      if (t >= total) break;
      const TcTile tile = walk.at(P, t);
      const bool tail = MODE == kDw && (tile.row_end - tile.row0) % 16 != 0;
      for (int j = 0; j < tile.steps; ++j) {
        if (!__all_sync(0xffffffffu, group_wait<false>(bar_empty(stage), phase ^ 1, abort_flag, P.wait_ns))) { ok = false; break; }
        if (elect_one()) {
          const uint32_t a = sbase + stage * stage_bytes, b = a + kGABytes;
          uint32_t bar = bar_full(stage);
          if constexpr (PAIR) {
            // one barrier of the leader counts the bytes of both CTAs; a step that is cleaned first is counted by each CTA
            if (tail && j == tile.steps - 1) {
              if (rank != 0) bar = bar_tail(stage);
              mbar_arrive_expect_tx(bar, stage_bytes);
            } else {
              if (rank == 0) mbar_arrive_expect_tx(bar, 2 * stage_bytes);
              else bar = map_to_rank(bar, 0);
            }
          } else {
            mbar_arrive_expect_tx(bar, stage_bytes);
          }
          const int k = j * kGK, n0 = tile.n0 + rank * b_columns;
          if (MODE == kDw) {
            for (int h = 0; h < 2; ++h) tma_2d<PAIR>(a + h * kGBlock, &map_a, tile.m0 + rank * kGRows + h * 64, tile.row0 + k, bar);
            for (int h = 0; h < P.b_bytes / kGBlock; ++h) tma_2d<PAIR>(b + h * kGBlock, &map_b, n0 + h * 64, tile.row0 + k, bar);
          } else {
            tma_2d<PAIR>(a, &map_a, k, tile.row0 + rank * kGRows, bar);
            if (MODE == kForward) {
              for (int h = 0; h < P.b_bytes / kGBlock; ++h) tma_3d<PAIR>(b + h * kGBlock, &map_b, n0 + h * 64, k, tile.expert, bar);
            } else {
              tma_3d<PAIR>(b, &map_b, k, n0, tile.expert, bar);
            }
          }
        }
        __syncwarp();
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // =========================== MMAs (a pair: by the leader) ===========================
    // rows [depth, 16 ks) of a last step belong to the next group: a reduction row is one 128-byte line of every box
    auto clean = [&](int stage, int depth, int ks) {
      const int lines = ks * 16 - depth, boxes = 2 + P.b_bytes / kGBlock;
      for (int i = lane; i < boxes * lines * 8; i += 32) {
        const int box = i / (lines * 8), q = i % (lines * 8);
        *reinterpret_cast<uint4 *>(smem + stage * stage_bytes + box * kGBlock + (depth + q / 8) * 128 + (q % 8) * 16) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async;" ::: "memory");
      __syncwarp();
    };
    int stage = 0, phase = 0, tile_i = 0;
    uint32_t acc_phase = 0, tail_phase = 0;      // tail_phase: parity of every stage's tail / clean barrier
    bool ok = true;
    if (rank == 0) {
      for (; ok && tile_i < rounds; ++tile_i) {
        const int t = round_tile(tile_i, me, G);
        if (t >= total) break;
        const TcTile tile = walk.at(P, t);
        const int b = tile_i & 1;
        // (the whole warp leaves together: lanes may see the abort flag at different times)
        const bool free_acc = PAIR ? group_wait<true>(bar_acc_empty(b), ((acc_phase >> b) & 1u) ^ 1u, abort_flag, P.wait_ns)
                                   : group_wait<false>(bar_acc_empty(b), ((acc_phase >> b) & 1u) ^ 1u, abort_flag, P.wait_ns);
        if (!__all_sync(0xffffffffu, free_acc)) break;
        acc_phase ^= 1u << b;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + b * P.acc_stride;
        const int length = MODE == kDw ? tile.row_end - tile.row0 : P.k_channels;
        for (int j = 0; j < tile.steps; ++j) {
          if (!__all_sync(0xffffffffu, group_wait<false>(bar_full(stage), phase, abort_flag, P.wait_ns))) { ok = false; break; }
          const uint32_t sa = sbase + stage * stage_bytes, sb = sa + kGABytes;
          const int left = length - j * kGK, depth = left < kGK ? left : kGK, ks = (depth + 15) / 16;
          if (MODE == kDw && depth < ks * 16) {
            clean(stage, depth, ks);
            if (PAIR) {
              if (!__all_sync(0xffffffffu, group_wait<true>(bar_clean(stage), (tail_phase >> stage) & 1u, abort_flag, P.wait_ns))) { ok = false; break; }
              tail_phase ^= 1u << stage;
            }
          }
          __syncwarp();
          if (elect_one()) {
            const uint64_t a_desc = MODE == kDw ? smem_desc_mn_sw128(sa) : smem_desc_k_sw128(sa);
            const uint64_t b_desc = MODE == kDx ? smem_desc_k_sw128(sb) : smem_desc_mn_sw128(sb);
            // 16 steps of the reduction: 32 bytes further in a K-major row, 16 lines further in the other layout
            constexpr uint32_t kA = MODE == kDw ? 2048 >> 4 : 32 >> 4, kB = MODE == kDx ? 32 >> 4 : 2048 >> 4;
            if (ks == 4) {
#pragma unroll
              for (int s = 0; s < 4; ++s) group_mma<PAIR>(d_tmem, a_desc + s * kA, b_desc + s * kB, P.idesc, (j | s) != 0);
            } else {
              for (int s = 0; s < ks; ++s) group_mma<PAIR>(d_tmem, a_desc + s * kA, b_desc + s * kB, P.idesc, (j | s) != 0);
            }
            group_commit<PAIR>(bar_empty(stage));
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (elect_one()) group_commit<PAIR>(bar_acc_full(b));
        __syncwarp();
      }
    } else if (MODE == kDw) {
      // follower: cleans its rows of every last step and tells the leader
      for (; ok && tile_i < rounds; ++tile_i) {
        const int t = round_tile(tile_i, me, G);
        if (t >= total) break;
        const TcTile tile = walk.at(P, t);
        const int length = tile.row_end - tile.row0, depth = length - (tile.steps - 1) * kGK, ks = (depth + 15) / 16;
        if (length % 16 != 0) {
          const int s = (stage + tile.steps - 1) % stages;
          if (!__all_sync(0xffffffffu, group_wait<false>(bar_tail(s), (tail_phase >> s) & 1u, abort_flag, tile_limit(P.wait_ns, tile.steps)))) break;
          tail_phase ^= 1u << s;
          clean(s, depth, ks);
          if (lane == 0) mbar_arrive_cluster(map_to_rank(bar_clean(s), 0));
        }
        stage = (stage + tile.steps) % stages;
      }
    }
  } else if (warp >= kGFirstEpilogueWarp) {
    // =========================== epilogue ===========================
    const int q = warp & 3, part = (warp - kGFirstEpilogueWarp) >> 2;
    const int width = P.bn / 4;                      // columns of this warp: a multiple of 16, at most 64
    float *bias_s = reinterpret_cast<float *>(smem + P.off_bias) + (warp - kGFirstEpilogueWarp) * 64;
    const bool relu = MODE == kForward && P.relu;
    unsigned char *stage_ptr = smem + P.off_stage + (warp - kGFirstEpilogueWarp) * P.box_cols * 64;
    int bias_at = -1;                                // what bias_s holds: expert * n_tiles + column tile
    uint32_t acc_phase = 0;
    for (int tile_i = 0; tile_i < rounds; ++tile_i) {
      const int t = round_tile(tile_i, me, G);
      if (t >= total) break;
      const TcTile tile = walk.at(P, t);
      const int b = tile_i & 1;
      const int m = (MODE == kDw ? tile.m0 : tile.row0) + rank * kGRows + q * 32 + lane, m_end = MODE == kDw ? P.m_channels : tile.row_end;
      const int col = tile.n0 + part * width;
      const int valid = m < m_end ? P.n_channels - col : 0;      // columns of this row that exist (a unit of 8 may reach into the pitch)
      const float *bias = nullptr;
      if (MODE == kForward && P.bias) {
        const int at = tile.expert * P.n_tiles + tile.n0 / P.bn;
        if (at != bias_at) {
          bias_at = at;
          const T *src = static_cast<const T *>(P.bias) + static_cast<int64_t>(tile.expert) * P.n_channels + col;
          __syncwarp();
          for (int i = lane; i < width; i += 32) bias_s[i] = col + i < P.n_channels ? to_f32(src[i]) : 0.f;
          __syncwarp();
        }
        bias = bias_s;
      }
      if (!__all_sync(0xffffffffu, group_wait<false>(bar_acc_full(b), (acc_phase >> b) & 1u, abort_flag, tile_limit(P.wait_ns, tile.steps)))) break;
      acc_phase ^= 1u << b;
      tc_fence_after();
      const uint32_t taddr = tmem_base + b * P.acc_stride + (static_cast<uint32_t>(q * 32) << 16) + part * width;
      const int64_t out_row = MODE == kDw ? static_cast<int64_t>(tile.expert) * P.m_channels + m : m;
      T *dst = static_cast<T *>(P.out) + out_row * P.out_pitch + col;
      float *dst_partial = MODE == kDw ? P.partial + (static_cast<int64_t>(tile.unit) * P.m_channels + m) * P.out_pitch + col : nullptr;
      uint32_t bits[2] = {0, 0};
      const int m_warp = m - lane;
      const bool by_tma = MODE != kDw && P.box_cols != 0 && m_warp + 32 <= m_end;     // (rows of the next group are not ours to write)
      // columns [c0, c0 + W) of this warp; `last`: the block they belong to is complete
      auto emit = [&](auto &r, int c0, uint32_t &word, bool last) {
        constexpr int W = sizeof(r) / 4;
        if (MODE == kDw && tile.steps == 0) {
#pragma unroll
          for (int i = 0; i < W; ++i) r[i] = 0;
        }
        if (MODE == kDw && P.piece) {
          if (c0 < valid) store_partial<W>(r, dst_partial + c0, valid - c0);
          __syncwarp();
          return;
        }
        uint4 v[W / 8];
        if (relu) convert_columns<T, W, true>(r, bias ? bias + c0 : nullptr, P.mask != nullptr, v, word);
        else convert_columns<T, W, false>(r, bias ? bias + c0 : nullptr, false, v, word);
        if (!by_tma) {
          if (c0 < valid) store_units<T, W / 8>(v, dst + c0, valid - c0);
          __syncwarp();
          return;
        }
        if (P.box_cols == 32) {      // 64-byte swizzle: unit u of row r lies at unit u ^ (r / 2 % 4)
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
#pragma unroll
          for (int u = 0; u < W / 8; ++u) *reinterpret_cast<uint4 *>(stage_ptr + lane * 64 + 16 * (u ^ ((lane >> 1) & 3))) = v[u];
        } else {                     // 96-byte rows as they are
          if (c0 == 0) {
            if (lane == 0) tma_store_wait_read();
            __syncwarp();
          }
#pragma unroll
          for (int u = 0; u < W / 8; ++u) *reinterpret_cast<uint4 *>(stage_ptr + lane * 96 + 2 * c0 + 16 * u) = v[u];
        }
        if (last) {
          fence_proxy_async();
          __syncwarp();
          const int x = P.box_cols == 32 ? col + c0 : col;
          if (lane == 0 && x < P.n_channels) tma_store_2d(&map_out, smem_u32(stage_ptr), x, m_warp);
        }
      };
#pragma unroll
      for (int piece = 0; piece < 2; ++piece) {
        const int c0 = 32 * piece;
        if (width - c0 >= 32) {
          uint32_t r[32];
          tmem_ld_32x32(taddr + c0, r);
          tmem_ld_wait();
          emit(r, c0, bits[piece], P.box_cols == 32);
        } else if (width - c0 == 16) {
          uint32_t r[16];
          tmem_ld_32x16(taddr + c0, r);
          tmem_ld_wait();
          emit(r, c0, bits[piece], true);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_cluster(map_to_rank(bar_acc_empty(b), 0));
        else mbar_arrive(bar_acc_empty(b));
      }
      if (MODE == kForward && P.mask && valid > 0) {
        unsigned char *line = P.mask + static_cast<int64_t>(m) * P.mask_pitch + col / 8;
        if (width == 64 && (reinterpret_cast<uintptr_t>(line) & 7) == 0 && valid > 32) {
          *reinterpret_cast<uint2 *>(line) = make_uint2(bits[0], bits[1]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * i < width && 16 * i < valid) *reinterpret_cast<uint16_t *>(line + 2 * i) = static_cast<uint16_t>(bits[i / 2] >> (16 * (i & 1)));
        }
      }
    }
    if (MODE != kDw && lane == 0) tma_store_wait_all();
  } else if (warp == 3 && MODE != kDw) {
    // rows of no group are zero
    T *out = static_cast<T *>(P.out);
    const int64_t width = P.out_pitch / 8, before = rows[0] * width, behind = static_cast<int64_t>(P.n - rows[P.experts]) * width;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + lane; i < before + behind; i += static_cast<int64_t>(gridDim.x) * 32)
      reinterpret_cast<uint4 *>(out)[i < before ? i : rows[P.experts] * width + i - before] = make_uint4(0, 0, 0, 0);
  }

  // =========================== teardown ===========================
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // a bounded wait expired: report, give copies in flight time to land, then release the tensor memory
    if (tid == 0 && P.status) atomicExch(P.status, 1);
    const unsigned long long t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) { }
    __syncthreads();
  }
  if (PAIR) cluster_sync();      // nobody leaves while the other CTA still signals its barriers or uses its memory
  if (warp == 1) {
    tc_fence_after();
    group_tmem_dealloc<PAIR>(tmem_base, P.tmem_cols);
  }
}

typedef CUresult (*GroupedEncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                    const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static GroupedEncodeFn grouped_encode_fn() {
  static GroupedEncodeFn fn = nullptr;
  if (fn == nullptr) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<GroupedEncodeFn>(p);
  }
  return fn;
}

// [n][channels] rows (stride in elements) or [experts][c_in][c_out] weights; boxes of 64 channels x box_rows, zeros outside
// (for stores: 32 channels with the 64-byte swizzle, or 48 without one).
static int encode_map(CUtensorMap *map, int dtype, const void *p, int rank, int64_t channels, int64_t rows, int64_t row_stride, int64_t outer, int box_rows,
                      int box_cols = 64) {
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(channels), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_stride) * 2, static_cast<cuuint64_t>(row_stride) * rows * 2};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = grouped_encode_fn()(map, dtype == SPIRA_B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                                         const_cast<void *>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                         box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : box_cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SPIRA_B200_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
  return SPIRA_B200_OK;
}

bool grouped_tc_rows_ok(const void *p, int64_t stride, int channels, int64_t n) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (n == 1 || (stride % 8 == 0 && stride >= channels));
}
bool grouped_tc_available() { return grouped_encode_fn() != nullptr; }

// Columns per tile: as few tiles of at most 256 as the width needs, of equal size in whole
// units of 64; when the tiles would not fill the SMs (few rows), narrower ones.
static int columns_per_tile(int channels, int64_t units) {
  int64_t tiles = div_up(channels, kGMaxN);
  while (tiles * units < sm_count() && div_up(channels, 2 * tiles) >= 64) tiles *= 2;
  return static_cast<int>(div_up(div_up(channels, tiles), 64) * 64);
}

int grouped_tc_dw_tiles(int c_in, int c_out) {
  return static_cast<int>(div_up(c_in, kGRows) * div_up(c_out, columns_per_tile(c_out, int64_t(1) << 30)));
}

// Two CTAs per tile where it has the rows and columns for both, enough work to fill the SMs in pairs and a reduction long
// enough for the fuller pipeline to matter.  Measured pair / single: 80 026 rows in 16 groups, 512 -> 2048: forward 146 /
// 155 us, dx 111 / 131 us, dW 127 / 147 us; 40 000 rows in 8 groups, 256 -> 1024: forward 62 / 44 us.
bool grouped_tc_pair(int mode, const spira_b200_grouped_desc &D) {
  if (mode == kDw) return D.c_in > kGRows && D.c_out >= 128 && D.n / D.experts >= 256;
  const int n = mode == kForward ? D.c_out : D.c_in, k = mode == kForward ? D.c_in : D.c_out;
  return n >= 128 && k >= 384 && D.n / D.experts >= 512 && D.n / 256 * div_up(n, kGMaxN) >= sm_count() / 2;
}

int grouped_tc_run(int mode, const spira_b200_grouped_desc &D, int w_pitch, int out_pitch, int piece, float *partial, int32_t *status, unsigned long long wait_ns, cudaStream_t st) {
  GroupedTcParams P{};
  P.offsets = D.offsets;
  P.partial = partial;
  P.status = status;
  P.n = static_cast<int>(D.n);
  P.experts = D.experts;
  P.piece = piece;
  P.wait_ns = wait_ns;
  P.out_pitch = out_pitch;
  const bool pair = grouped_tc_pair(mode, D);
  P.tile_rows = pair ? 2 * kGRows : kGRows;
  int64_t units;
  if (mode == kDw) {
    P.out = D.dweight;
    P.m_channels = D.c_in;
    P.n_channels = D.c_out;
    P.m_tiles = static_cast<int>(div_up(D.c_in, P.tile_rows));
    units = (piece ? group_tiles_bound(D.n, D.experts, piece) : D.experts) * P.m_tiles;
    P.bn = columns_per_tile(D.c_out, int64_t(1) << 30);
  } else {
    P.out = mode == kForward ? D.y : D.dx;
    P.bias = mode == kForward ? D.bias : nullptr;
    P.relu = mode == kForward ? D.relu : 0;
    P.mask = mode == kForward ? static_cast<unsigned char *>(D.mask) : nullptr;
    P.mask_pitch = mask_pitch(D.c_out);
    P.n_channels = mode == kForward ? D.c_out : D.c_in;
    P.k_channels = mode == kForward ? D.c_in : D.c_out;
    P.m_tiles = 1;
    units = group_tiles_bound(D.n, D.experts, P.tile_rows);
    P.bn = columns_per_tile(P.n_channels, pair ? int64_t(1) << 30 : units);
  }
  if (pair) P.bn = static_cast<int>(div_up(P.bn, 128) * 128);      // (each CTA holds half of the columns in 64-wide boxes)
  P.n_tiles = static_cast<int>(div_up(P.n_channels, P.bn));
  const bool b_n_major = mode != kDx;
  const int b_columns = pair ? P.bn / 2 : P.bn;
  P.b_bytes = b_columns * 128;             // (a multiple of 8 KB: whole boxes)
  P.acc_stride = 32;
  while (P.acc_stride < P.bn) P.acc_stride *= 2;
  P.tmem_cols = 2 * P.acc_stride;
  P.idesc = (1u << 4) | (D.dtype == SPIRA_B200_BF16 ? (1u << 7) | (1u << 10) : 0u) | (mode == kDw ? 1u << 15 : 0u) | (b_n_major ? 1u << 16 : 0u) |
            (static_cast<uint32_t>(P.bn >> 3) << 17) | (static_cast<uint32_t>(P.tile_rows >> 4) << 24);
  const int bars = 8 * (4 * kGMaxStages + 5);
  int fixed = kGBiasBytes + bars + 16 + 12 * (D.experts + 2);
  const int stage_bytes = kGABytes + P.b_bytes;
  // Stores: a scattered 16-byte store of 32 rows takes 32 passes of the load/store unit (4096 per tile of 128 x 256, where a
  // reduction step takes 512), so results of short reductions leave through shared memory and TMA.  Longer ones hide the
  // stores, and the staging buffers would cost a pipeline stage (80 026 x 2048 -> 512: 111 us direct, 121 us staged;
  // 254 726 x 96 -> 384: 75 us staged, 81 us direct).
  const int width = P.bn / 4, steps = static_cast<int>(div_up(P.k_channels, kGK));
  P.box_cols = mode == kDw || width == 16 || steps > 8 ? 0 : width == 48 ? 48 : 32;
  const int staging = kGEpilogueWarps * P.box_cols * 64;
  fixed += staging;
  P.stages = (kGSmemBudget - fixed) / stage_bytes;
  if (P.stages > kGMaxStages) P.stages = kGMaxStages;
  P.off_stage = P.stages * stage_bytes;
  P.off_bias = P.off_stage + staging;
  P.off_bar = P.off_bias + kGBiasBytes;
  P.off_groups = P.off_bar + bars + 8;
  const size_t smem = static_cast<size_t>(P.off_stage) + fixed + 1024;

  // A thread that has made no CUDA call yet (autograd's) has no current context, which the driver call below needs.
  int device = 0;
  SB_CHECK_CUDA(cudaGetDevice(&device));
  SB_CHECK_CUDA(cudaSetDevice(device));
  alignas(64) CUtensorMap map_a, map_b, map_out;
  int rc;
  const int64_t x_stride = D.n == 1 ? pitch8(D.c_in) : D.x_stride, dy_stride = D.n == 1 ? pitch8(D.c_out) : D.dy_stride;
  if (mode == kForward) {
    rc = encode_map(&map_a, D.dtype, D.x, 2, D.c_in, D.n, x_stride, 1, kGRows);
    if (rc == SPIRA_B200_OK) rc = encode_map(&map_b, D.dtype, D.weight, 3, D.c_out, D.c_in, w_pitch, D.experts, kGK);
  } else if (mode == kDx) {
    rc = encode_map(&map_a, D.dtype, D.dy, 2, D.c_out, D.n, dy_stride, 1, kGRows);
    if (rc == SPIRA_B200_OK) rc = encode_map(&map_b, D.dtype, D.weight, 3, D.c_out, D.c_in, w_pitch, D.experts, b_columns);
  } else {
    rc = encode_map(&map_a, D.dtype, D.x, 2, D.c_in, D.n, x_stride, 1, kGK);
    if (rc == SPIRA_B200_OK) rc = encode_map(&map_b, D.dtype, D.dy, 2, D.c_out, D.n, dy_stride, 1, kGK);
  }
  if (rc == SPIRA_B200_OK && P.box_cols) rc = encode_map(&map_out, D.dtype, P.out, 2, P.n_channels, D.n, P.out_pitch, 1, 32, P.box_cols);
  else map_out = map_a;
  if (rc != SPIRA_B200_OK) return rc;
  const int64_t tiles = units * P.n_tiles;
  SB_CHECK_ARG(tiles < (int64_t(1) << 31) - 65536, "grouped_linear: too many tiles");
  const int64_t workers = pair ? sm_count() / 2 : sm_count();
  const unsigned grid = static_cast<unsigned>(tiles < workers ? (tiles < 1 ? 1 : tiles) : workers) * (pair ? 2 : 1);
  auto go = [&](auto kernel) -> int {
    const int allowed = allow_smem(kernel, kGSmemBudget + 1024);      // (what `stages` is cut to)
    if (allowed != SPIRA_B200_OK) return allowed;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kGThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    if (pair) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = 2;
      attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
      ++cfg.numAttrs;
    }
    if (pdl_enabled()) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
      ++cfg.numAttrs;
    }
    cfg.attrs = attr;
    SB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, P, map_a, map_b, map_out));
    count_operator_launch();
    return SPIRA_B200_OK;
  };
  auto pick = [&](auto type) -> int {
    using T = decltype(type);
    if (pair) return mode == kForward ? go(grouped_tc_kernel<T, kForward, true>) : mode == kDx ? go(grouped_tc_kernel<T, kDx, true>) : go(grouped_tc_kernel<T, kDw, true>);
    return mode == kForward ? go(grouped_tc_kernel<T, kForward, false>) : mode == kDx ? go(grouped_tc_kernel<T, kDx, false>) : go(grouped_tc_kernel<T, kDw, false>);
  };
  return D.dtype == SPIRA_B200_F16 ? pick(__half{}) : pick(__nv_bfloat16{});
}

}  // namespace sb
