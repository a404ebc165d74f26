// Routing of rows to experts and moving them there and back.
//
//   route     the k experts of every row (the k largest logits), their weights, and the place of every (row, expert) pair
//             in expert order: a stable counting sort by expert
//   clear     rows of places that no slot names = 0 (before a dispatch)
//   dispatch  rows[slots[t][j]] = x[t]
//   combine   out[t] = sum_j weights[t][j] * rows[slots[t][j]]
//
// Every result is a function of the inputs alone: counts are integers, places follow from counts and ranks, sums run over
// j in order.  Dispatch and combine are bound by memory (127 363 x 96 fp16, k 2: 11 us = 6.8 TB/s there, 14 us = 5.3 TB/s
// back), routing by its two launches, the selection (127 363 x 64 fp16, k 4: 13 us) and the sort (11 us) for 24 MB, all of it
// by the launch for a few rows.
#include <atomic>
#include <cfloat>
#include <cmath>

#include "common.cuh"
#include "elem.cuh"

namespace sb {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 32;
constexpr int kRouteThreads = 1024;     // one CTA per SM: few histograms to add up (two CTAs of 512 threads: 26.6 instead of 23.2 us)
constexpr int kRouteWarps = kRouteThreads / 32;
static_assert(kRouteWarps == 32, "the warps' counts of an expert are added up by the lanes of one warp");
constexpr int kSmallRouteEntries = 4096;   // (row, expert) pairs up to which one CTA does everything in one launch

// Order of logits as unsigned numbers: -inf < ... < +inf < NaN, -0 = +0.  kGone (a number below every logit but equal to
// nothing) marks what is masked (-inf) or chosen already.
constexpr uint32_t kGone = 0;
__device__ __forceinline__ uint32_t logit_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == -INFINITY) return kGone;
  const uint32_t b = __float_as_uint(v + 0.f);   // -0 + 0 = +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  if (k == 0xffffffffu) return NAN;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 16-bit logits: order (16 bits) and expert (9 bits) make one number per expert, equal logits ordered by the lower index, so
// that a maximum takes one instruction per expert.  Adding +0 makes -0 equal to +0 and every NaN the positive one, which
// is then the largest; what is not above -inf counts as masked.
__device__ __forceinline__ uint32_t canonical2(uint32_t w, __half) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
  return r;
}
__device__ __forceinline__ uint32_t canonical2(uint32_t w, __nv_bfloat16) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
  return r;
}
template <typename T>
constexpr uint32_t kMinusInf16 = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
// the order of both halves of a word
template <typename T>
__device__ __forceinline__ uint32_t order2(uint32_t w) {
  w = canonical2(w, T{});
  const uint32_t negative = ((w >> 15) & 0x00010001u) * 0xffffu;
  return w ^ (negative | 0x80008000u);
}
// a logit from its order
template <typename T>
__device__ __forceinline__ float order_logit(uint32_t o) {
  const unsigned short h = static_cast<unsigned short>(o & 0x8000u ? o ^ 0x8000u : ~o);
  T v;
  *reinterpret_cast<unsigned short *>(&v) = h;
  return to_f32(v);
}
static_assert(kMaxExperts == 512, "the packed keys hold nine bits of expert");

// The packed keys of the experts [c0, c0 + EPL) of a row; experts that do not exist are masked.
template <typename T, int EPL>
__device__ __forceinline__ void load_packed(const T *row, int c0, int experts, bool live, bool vec_ok, uint32_t (&key)[EPL]) {
  uint32_t w[EPL / 2];
  if (live && vec_ok && c0 + EPL <= experts) {
    constexpr int V = EPL >= 8 ? 4 : EPL / 2;      // words per access
#pragma unroll
    for (int i = 0; i < EPL / 2; i += V) {
      const Vec<uint32_t, V> q = *reinterpret_cast<const Vec<uint32_t, V> *>(row + c0 + 2 * i);
#pragma unroll
      for (int j = 0; j < V; ++j) w[i + j] = q.v[j];
    }
  } else {
    const unsigned short *h = reinterpret_cast<const unsigned short *>(row + c0);
#pragma unroll
    for (int i = 0; i < EPL / 2; ++i) {
      const uint32_t lo = live && c0 + 2 * i < experts ? h[2 * i] : kMinusInf16<T>, hi = live && c0 + 2 * i + 1 < experts ? h[2 * i + 1] : kMinusInf16<T>;
      w[i] = lo | hi << 16;
    }
  }
#pragma unroll
  for (int i = 0; i < EPL / 2; ++i) {
    const uint32_t o = order2<T>(w[i]), tail = static_cast<uint32_t>(kMaxExperts - 1 - c0 - 2 * i);
    key[2 * i] = (o & 0xffffu) * 512u + tail;
    key[2 * i + 1] = (o >> 16) * 512u + tail - 1u;
  }
}

// EPL consecutive elements of a row from column c0 on as fp32, `fill` outside the row.
template <typename T, int EPL>
__device__ __forceinline__ void load_logits(const T *row, int c0, int experts, bool live, bool vec_ok, float fill, float (&v)[EPL]) {
  constexpr int V = EPL * sizeof(T) >= 16 ? 16 / sizeof(T) : EPL;
  if (live && vec_ok && c0 + EPL <= experts) {
#pragma unroll
    for (int i = 0; i < EPL; i += V) {
      float f[V];
      load_f32<T, V>(row + c0 + i, f);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i + j] = f[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = live && c0 + i < experts ? to_f32(row[c0 + i]) : fill;
  }
}

// The rows [r0, r1) of a CTA.  A row takes G neighbouring lanes with EPL consecutive experts each (G * EPL >= experts): few
// lanes with many experts keep the number of shuffles small (at 64 experts and k = 4, 4 lanes x 16 experts execute a
// quarter of the instructions of 32 lanes x 2).  Choices are collected in shared memory, so that results leave in whole
// lines and nothing is read back.
template <typename T, int G, int EPL>
__device__ __forceinline__ void route_rows(const T *logits, int64_t row_stride, int64_t r0, int64_t r1, int experts, int k, int renormalize,
                                           float *weights, int32_t *chosen, int *hist, int *stash) {
  constexpr int V = EPL * sizeof(T) >= 16 ? 16 / sizeof(T) : EPL;
  const bool vec_ok = reinterpret_cast<uintptr_t>(logits) % (V * sizeof(T)) == 0 && row_stride % V == 0;
  const int g = threadIdx.x & (G - 1), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kRows = kRouteThreads / G, kWarpRows = 32 / G;
  constexpr bool kPacked = sizeof(T) == 2;
  constexpr uint32_t kMaskedOrder = 0xffffu & ~kMinusInf16<T>;      // the order of -inf
  int *warp_e = stash + warp * kWarpRows * k * 2;                       // [rows of the warp][k]
  float *warp_w = reinterpret_cast<float *>(warp_e + kWarpRows * k);
  int *my_e = warp_e + lane / G * k;
  float *my_w = warp_w + lane / G * k;
  for (int64_t r = r0; r < r1; r += kRows) {
    const int64_t row = r + threadIdx.x / G;
    const bool live = row < r1;
    uint32_t key[EPL];
    if constexpr (kPacked) {
      load_packed<T, EPL>(logits + row * row_stride, g * EPL, experts, live, vec_ok, key);
    } else {
      float v[EPL];
      load_logits<T, EPL>(logits + row * row_stride, g * EPL, experts, live, vec_ok, -INFINITY, v);
#pragma unroll
      for (int i = 0; i < EPL; ++i) key[i] = logit_key(v[i]);
    }
    float top = 0.f, sum = 0.f, total = 0.f;
    uint32_t last = 0x80000000u;
    for (int j = 0; j < k; ++j) {
      uint32_t best = kGone;
      bool found;
      float logit;
      int e;
      if constexpr (kPacked) {
        // the largest key below the last one: differences wrap, what is not below it stays under 2^31
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < EPL; ++i) m = __viaddmax_u32(key[i], 0u - last, m);
#pragma unroll
        for (int d = 1; d < G; d *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d, G));
        last = m >= 0x80000000u ? m + last : 0;
        e = kMaxExperts - 1 - static_cast<int>(last & (kMaxExperts - 1));
        found = last >> 9 > kMaskedOrder;
        logit = order_logit<T>(last >> 9);
      } else {
        int at = 0;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (key[i] > best) { best = key[i]; at = i; }     // (strict: the lowest index of equal logits)
        e = g * EPL + at;
#pragma unroll
        for (int d = 1; d < G; d *= 2) {
          const uint32_t ob = __shfl_xor_sync(0xffffffffu, best, d, G);
          const int oe = __shfl_xor_sync(0xffffffffu, e, d, G);
          if (ob > best || (ob == best && oe < e)) { best = ob; e = oe; }
        }
      }
      if constexpr (!kPacked) {
        found = best != kGone;
        logit = key_logit(best);
      }
      if (j == 0) {
        top = found ? logit : 0.f;
        if (!renormalize) {      // the softmax runs over all experts: while every logit is still there
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            const bool there = kPacked ? key[i] >> 9 > kMaskedOrder : key[i] != kGone;
            if (there) total += expf((kPacked ? order_logit<T>(key[i] >> 9) : key_logit(key[i])) - top);
          }
#pragma unroll
          for (int d = 1; d < G; d *= 2) total += __shfl_xor_sync(0xffffffffu, total, d, G);
        }
      }
      if constexpr (!kPacked) {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (g * EPL + i == e) key[i] = kGone;
      }
      const float score = found ? expf(logit - top) : 0.f;
      sum += score;
      if (g == 0) {
        my_w[j] = score;
        my_e[j] = found ? e : -1;
        if (live && found) atomicAdd(hist + e, 1);
      }
    }
    __syncwarp();
    const float denom = renormalize ? sum : total;
    for (int j = g; j < k; j += G) my_w[j] = my_e[j] >= 0 ? my_w[j] / denom : 0.f;
    __syncwarp();
    const int64_t first = r + warp * kWarpRows;
    const int count = static_cast<int>(r1 - first < kWarpRows ? (r1 > first ? r1 - first : 0) : kWarpRows) * k;
    for (int i = lane; i < count; i += 32) {
      weights[first * k + i] = warp_w[i];
      chosen[first * k + i] = warp_e[i];
    }
    __syncwarp();
  }
}

// Places of the entries [n0, n1) (entry = row * k + j) of one CTA's rows.  Warps take consecutive pieces; a piece is counted
// first (which needs nothing of the other CTAs, so it overlaps the reads of their histograms: 127 363 x 64, k 4 19.2 us in
// all, 19.6 when counted behind them), then ranked 32 entries at a time.
struct Piece {
  int64_t begin, end;
  __device__ __forceinline__ Piece(int64_t n0, int64_t n1) {
    const int64_t piece = ((n1 - n0 + kRouteWarps * 32 - 1) / (kRouteWarps * 32)) * 32;
    const int warp = threadIdx.x >> 5;
    begin = n0 + piece * warp < n1 ? n0 + piece * warp : n1;
    end = begin + piece < n1 ? begin + piece : n1;
  }
};
constexpr int kPlaceBatch = 8;      // loads in flight

__device__ __forceinline__ void count_entries(const int32_t *chosen, int64_t n0, int64_t n1, int experts, int *warp_counts) {
  const int lane = threadIdx.x & 31;
  const Piece p(n0, n1);
  int *mine = warp_counts + (threadIdx.x >> 5) * (experts | 1);
  for (int e = lane; e < experts; e += 32) mine[e] = 0;
  __syncwarp();
  for (int64_t i = p.begin; i < p.end; i += 32 * kPlaceBatch) {
    int e[kPlaceBatch];
#pragma unroll
    for (int q = 0; q < kPlaceBatch; ++q) e[q] = i + 32 * q + lane < p.end ? chosen[i + 32 * q + lane] : -1;
#pragma unroll
    for (int q = 0; q < kPlaceBatch; ++q)
      if (e[q] >= 0) atomicAdd(mine + e[q], 1);
  }
}

// `base[e]`: the place of the CTA's first entry of expert e
__device__ __forceinline__ void place_entries(const int32_t *chosen, int64_t n0, int64_t n1, int experts, const int *base, int *warp_base,
                                              int32_t *slots, int32_t *order) {
  constexpr int kBatch = kPlaceBatch;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Piece p(n0, n1);
  const int64_t p0 = p.begin, p1 = p.end;
  const int pitch = experts | 1;                // (odd: the counts of one expert lie in different banks)
  int *mine = warp_base + warp * pitch;
  for (int e = warp; e < experts; e += kRouteWarps) {      // lane w: the first place of warp w
    int *at = warp_base + lane * pitch + e;
    const int own = *at;
    int sum = own;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    *at = base[e] + sum - own;
  }
  __syncthreads();
  for (int64_t i0 = p0; i0 < p1; i0 += 32 * kBatch) {
    int batch[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) batch[q] = i0 + 32 * q + lane < p1 ? chosen[i0 + 32 * q + lane] : -1;
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int64_t i = i0 + 32 * q;
      if (i >= p1) break;
      const int e = batch[q];
      const uint32_t peers = __match_any_sync(0xffffffffu, e);
      const int rank = __popc(peers & ((1u << lane) - 1u));
      int slot = -1;
      if (e >= 0) slot = mine[e] + rank;
      __syncwarp();
      if (e >= 0 && rank == 0) mine[e] += __popc(peers);
      __syncwarp();
      if (i + lane < p1) {
        slots[i + lane] = slot;
        if (slot >= 0) order[slot] = static_cast<int32_t>(i + lane);
      }
    }
  }
}

// Exclusive prefix of totals[0..experts) into first[0..experts] by one warp.
__device__ __forceinline__ void scan_experts(const int *totals, int *first, int experts) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    int v = e0 + lane < experts ? totals[e0 + lane] : 0;
    const int own = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    if (e0 + lane < experts) first[e0 + lane] = run + v - own;
    run += __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) first[experts] = run;
}

struct RouteParams {
  const void *logits;
  int64_t n, row_stride, rows_per_cta;
  int experts, k, renormalize;
  float *weights;
  int32_t *chosen, *slots, *order, *offsets;
  int *block_hist;      // [CTAs][experts]
};

// Few rows: everything in one CTA and one launch.
template <typename T, int G, int EPL>
__global__ void __launch_bounds__(kRouteThreads) route_small_kernel(const RouteParams P) {
  extern __shared__ int route_smem[];
  int *hist = route_smem, *first = hist + P.experts, *warp_base = first + P.experts + 1, *stash = warp_base + kRouteWarps * (P.experts | 1);
  pdl_trigger();
  for (int e = threadIdx.x; e < P.experts; e += kRouteThreads) hist[e] = 0;
  pdl_wait();
  __syncthreads();
  route_rows<T, G, EPL>(static_cast<const T *>(P.logits), P.row_stride, 0, P.n, P.experts, P.k, P.renormalize, P.weights, P.chosen, hist, stash);
  __syncthreads();
  count_entries(P.chosen, 0, P.n * P.k, P.experts, warp_base);
  if (threadIdx.x < 32) scan_experts(hist, first, P.experts);
  __syncthreads();
  place_entries(P.chosen, 0, P.n * P.k, P.experts, first, warp_base, P.slots, P.order);
  for (int e = threadIdx.x; e <= P.experts; e += kRouteThreads) P.offsets[e] = first[e];
  for (int64_t i = first[P.experts] + threadIdx.x; i < P.n * P.k; i += kRouteThreads) P.order[i] = -1;
}

template <typename T, int G, int EPL>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteParams P) {
  extern __shared__ int route_smem[];
  pdl_trigger();
  for (int e = threadIdx.x; e < P.experts; e += kRouteThreads) route_smem[e] = 0;
  pdl_wait();
  __syncthreads();
  const int64_t r0 = blockIdx.x * P.rows_per_cta, r1 = r0 + P.rows_per_cta < P.n ? r0 + P.rows_per_cta : P.n;
  route_rows<T, G, EPL>(static_cast<const T *>(P.logits), P.row_stride, r0, r1, P.experts, P.k, P.renormalize, P.weights, P.chosen, route_smem,
                        route_smem + P.experts);
  __syncthreads();
  for (int e = threadIdx.x; e < P.experts; e += kRouteThreads) P.block_hist[static_cast<int64_t>(blockIdx.x) * P.experts + e] = route_smem[e];
}

// Every CTA adds up the histograms by itself (CTAs x experts numbers from L2) instead of waiting for a scan launch.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteParams P) {
  extern __shared__ int route_smem[];
  int *totals = route_smem, *before = totals + P.experts, *first = before + P.experts, *warp_base = first + P.experts + 1;
  pdl_trigger();
  for (int e = threadIdx.x; e < P.experts; e += kRouteThreads) totals[e] = before[e] = 0;
  pdl_wait();
  __syncthreads();
  const int64_t r0 = blockIdx.x * P.rows_per_cta, r1 = r0 + P.rows_per_cta < P.n ? r0 + P.rows_per_cta : P.n;
  count_entries(P.chosen, r0 * P.k, r1 * P.k, P.experts, warp_base);
  const int G = gridDim.x;
  // W neighbouring experts per thread (16-byte reads where the count allows), all CTAs spread over the threads
  auto add_up = [&](auto width) {
    constexpr int W = decltype(width)::value;
    const int groups = P.experts / W, lanes = groups < kRouteThreads ? kRouteThreads / groups : 1;
    for (int i = threadIdx.x; i < groups * lanes; i += kRouteThreads) {
      const int e = i % groups * W;
      int all[W] = {}, mine[W] = {};
#pragma unroll 8
      for (int b = i / groups; b < G; b += lanes) {
        const Vec<int, W> c = *reinterpret_cast<const Vec<int, W> *>(P.block_hist + static_cast<int64_t>(b) * P.experts + e);
#pragma unroll
        for (int q = 0; q < W; ++q) {
          all[q] += c.v[q];
          if (b < static_cast<int>(blockIdx.x)) mine[q] += c.v[q];
        }
      }
#pragma unroll
      for (int q = 0; q < W; ++q) {
        atomicAdd(totals + e + q, all[q]);
        if (mine[q]) atomicAdd(before + e + q, mine[q]);
      }
    }
  };
  if (P.experts % 4 == 0) add_up(std::integral_constant<int, 4>{});
  else add_up(std::integral_constant<int, 1>{});
  __syncthreads();
  if (threadIdx.x < 32) scan_experts(totals, first, P.experts);
  __syncthreads();
  for (int e = threadIdx.x; e < P.experts; e += kRouteThreads) before[e] += first[e];
  __syncthreads();
  place_entries(P.chosen, r0 * P.k, r1 * P.k, P.experts, before, warp_base, P.slots, P.order);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= P.experts; e += kRouteThreads) P.offsets[e] = first[e];
  const int64_t total = P.n * P.k;
  for (int64_t i = first[P.experts] + static_cast<int64_t>(blockIdx.x) * kRouteThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(G) * kRouteThreads)
    P.order[i] = -1;
}

// dlogits: with u_j = dweights of the chosen experts and dot = sum_j u_j w_j,
//   softmax over the chosen:  d[e_j] = w_j (u_j - dot), 0 elsewhere
//   softmax over all:         d[e] = p_e ([e chosen] u_e - dot),  p_e = exp(l_e - max) / sum
template <typename T, int G, int EPL>
__global__ void __launch_bounds__(256) route_backward_kernel(const T *logits, int64_t n, int64_t row_stride, int experts, int k, int renormalize,
                                                             const float *weights, const int32_t *chosen, const float *dweights,
                                                             int64_t dw_row, int64_t dw_col, T *dlogits) {
  pdl_trigger();
  pdl_wait();
  constexpr int V = EPL * sizeof(T) >= 16 ? 16 / sizeof(T) : EPL;
  const bool vec_ok = reinterpret_cast<uintptr_t>(logits) % (V * sizeof(T)) == 0 && row_stride % V == 0;
  const bool out_ok = reinterpret_cast<uintptr_t>(dlogits) % (V * sizeof(T)) == 0 && experts % V == 0;
  const int g = threadIdx.x & (G - 1);
  constexpr int kRows = 256 / G;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / G;
  const bool live = row < n;
  float v[EPL], d[EPL];
  if (!renormalize) load_logits<T, EPL>(logits + row * row_stride, g * EPL, experts, live, vec_ok, -INFINITY, v);
  float dot = 0.f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) d[i] = 0.f;
  for (int j0 = 0; j0 < k; j0 += G) {           // lane g brings entry j0 + g, then everybody sees all of them
    const int j = j0 + g;
    const bool there = live && j < k;
    const int e = there ? chosen[row * k + j] : -1;
    const float u = e >= 0 ? dweights[row * dw_row + j * dw_col] : 0.f, w = e >= 0 ? weights[row * k + j] : 0.f;
    float part = e >= 0 ? u * w : 0.f;
#pragma unroll
    for (int s = 1; s < G; s *= 2) part += __shfl_xor_sync(0xffffffffu, part, s, G);
    dot += part;
    const int stop = k - j0 < G ? k - j0 : G;
    for (int q = 0; q < stop; ++q) {
      const int eq = __shfl_sync(0xffffffffu, e, q, G);
      const float uq = __shfl_sync(0xffffffffu, u, q, G);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (eq == g * EPL + i) d[i] = uq;
    }
  }
  // (renormalize: the places of the chosen are found a second time, now that the dot product is known)
  if (renormalize) {
    float r[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) r[i] = 0.f;
    for (int j0 = 0; j0 < k; j0 += G) {
      const int j = j0 + g;
      const int e = live && j < k ? chosen[row * k + j] : -1;
      const float w = e >= 0 ? weights[row * k + j] : 0.f;
      const int stop = k - j0 < G ? k - j0 : G;
      for (int q = 0; q < stop; ++q) {
        const int eq = __shfl_sync(0xffffffffu, e, q, G);
        const float wq = __shfl_sync(0xffffffffu, w, q, G);
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (eq == g * EPL + i) r[i] = wq * (d[i] - dot);
      }
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = r[i];
  } else {
    float top = -INFINITY, total = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      nan |= v[i] != v[i];
      top = fmaxf(top, v[i]);
    }
#pragma unroll
    for (int s = 1; s < G; s *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s, G));
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      v[i] = v[i] == -INFINITY ? 0.f : expf(v[i] - top);
      total += v[i];
    }
    if (nan) total = NAN;
#pragma unroll
    for (int s = 1; s < G; s *= 2) total += __shfl_xor_sync(0xffffffffu, total, s, G);
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = v[i] == 0.f ? 0.f : v[i] / total * (d[i] - dot);
  }
  if (!live) return;
  T *out = dlogits + row * experts + g * EPL;
  if (out_ok && (g + 1) * EPL <= experts) {
#pragma unroll
    for (int i = 0; i < EPL; i += V) {
      float f[V];
#pragma unroll
      for (int q = 0; q < V; ++q) f[q] = d[i + q];
      store_f32<T, V>(out + i, f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (g * EPL + i < experts) out[i] = from_f32<T>(d[i]);
  }
}

// ------------------------------------------------------------------------------------------------ rows to experts and back
// A thread moves V elements of one row; the threads of a row are neighbours, so reads and writes are whole lines whatever
// order the places come in.  Row indices outside [0, rows) are skipped (they come from memory, not from the host).
struct MoveParams {
  const void *x, *y;
  const float *weights;
  const int32_t *slots, *offsets, *order;
  void *out;
  float *dweights;
  int64_t n, x_stride, y_stride, w_row, w_col;
  int channels, k, experts;
  int clear, clear_here;             // rows of places that no slot names are cleared / by the one CTA that writes the rows
  int64_t rows_per_launch_row;       // rows of one blockIdx.y: rows * pieces stays below 2^31
  uint64_t div_mul;                  // i / pieces = (i * div_mul) >> div_shift for 0 <= i < 2^31
  int div_shift;
};

template <typename T, int V>
__device__ __forceinline__ void zero_tail(const MoveParams &P, T *rows, int vecs) {
  const int64_t total = P.n * P.k;
  int64_t tail = P.offsets[P.experts];
  tail = tail < 0 ? 0 : tail > total ? total : tail;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * gridDim.y * blockDim.x, work = (total - tail) * vecs;
  const float zero[V] = {};
  for (int64_t i = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x; i < work; i += threads)
    store_f32<T, V>(rows + (tail + i / vecs) * P.channels + (i % vecs) * V, zero);
}

// Zeros for the places that no slot names, before the rows are written: `order` says which pair a place belongs to, and a place
// whose pair says the same needs nothing.  All others get zeros, so whatever `order` holds (it may be older than the
// slots, or absent) costs writes and never a wrong row.  A warp looks at 32 places, whose rows are neighbours.
template <int BYTES>
__device__ __forceinline__ void clear_places(const int32_t *slots, const int32_t *order, int64_t total, int64_t row_bytes, unsigned char *rows, int64_t p0) {
  typedef typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 4, uint32_t, unsigned short>::type>::type Word;
  const int lane = threadIdx.x & 31;
  const int64_t p = p0 + lane;
  bool named = p >= total;
  if (!named && order) {
    const int32_t pair = order[p];
    named = pair >= 0 && pair < total && slots[pair] == p;
  }
  uint32_t open = __ballot_sync(0xffffffffu, !named);
  const int64_t words = row_bytes / BYTES;
  if (open == 0xffffffffu) {
    Word *at = reinterpret_cast<Word *>(rows + p0 * row_bytes);
    for (int64_t i = lane; i < 32 * words; i += 32) at[i] = Word{};
    return;
  }
  for (; open != 0; open &= open - 1) {
    Word *at = reinterpret_cast<Word *>(rows + (p0 + __ffs(open) - 1) * row_bytes);
    for (int64_t i = lane; i < words; i += 32) at[i] = Word{};
  }
}

// In a launch of its own (bound by two dependent loads: 3.5 us for 254 726 places), or, where the rows are written by one CTA,
// in that CTA (few rows: dispatch 9.7 us at the host, 12.1 with two launches).
template <int BYTES>
__global__ void __launch_bounds__(256) clear_kernel(const int32_t *slots, const int32_t *order, int64_t total, int64_t row_bytes, unsigned char *rows) {
  pdl_trigger();
  pdl_wait();
  clear_places<BYTES>(slots, order, total, row_bytes, rows, (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) & ~static_cast<int64_t>(31));
}
template <typename T, int V>
__device__ __forceinline__ void clear_here(const MoveParams &P) {
  const int64_t total = P.n * P.k;
  for (int64_t p0 = threadIdx.x & ~31u; p0 < total; p0 += 256)
    clear_places<V * static_cast<int>(sizeof(T))>(P.slots, P.order, total, P.channels * static_cast<int64_t>(sizeof(T)), static_cast<unsigned char *>(P.out), p0);
  __syncthreads();
}

// The row and the first channel of a thread; false behind the last row.
template <int V>
__device__ __forceinline__ bool my_piece(const MoveParams &P, int64_t &row, int &c) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const uint32_t r = static_cast<uint32_t>((i * P.div_mul) >> P.div_shift);
  row = static_cast<int64_t>(blockIdx.y) * P.rows_per_launch_row + r;
  c = static_cast<int>(i - r * static_cast<uint32_t>(P.channels / V)) * V;
  return r < P.rows_per_launch_row && row < P.n;
}

// K: experts per row, 0 = P.k.  The places of a row are known before its first load, all K copies are in flight together.
template <typename T, int V, int K>
__global__ void __launch_bounds__(256) dispatch_kernel(const MoveParams P) {
  pdl_trigger();
  pdl_wait();
  if (P.clear_here) clear_here<T, V>(P);
  const int64_t total = P.n * P.k;
  T *rows = static_cast<T *>(P.out);
  int64_t row;
  int c;
  if (my_piece<V>(P, row, c)) {
    const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(P.x) + row * P.x_stride + c);
    const int k = K ? K : P.k;
#pragma unroll
    for (int j = 0; j < k; ++j) {
      const int64_t slot = P.slots[row * k + j];
      if (slot >= 0 && slot < total) *reinterpret_cast<Vec<T, V> *>(rows + slot * P.channels + c) = v;
    }
  }
  if (P.offsets) zero_tail<T, V>(P, rows, P.channels / V);
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(256) combine_kernel(const MoveParams P) {
  pdl_trigger();
  pdl_wait();
  const int64_t total = P.n * P.k;
  const T *rows = static_cast<const T *>(P.y);
  int64_t row;
  int c;
  if (!my_piece<V>(P, row, c)) return;
  constexpr int B = K && K < 4 ? K : 4;          // rows on their way at a time
  const int k = K ? K : P.k;
  float acc[V] = {};
#pragma unroll
  for (int j0 = 0; j0 < k; j0 += B) {
    Vec<T, V> v[B];
    float w[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int64_t slot = j0 + j < k ? P.slots[row * k + j0 + j] : -1;
      w[j] = j0 + j < k && P.weights ? P.weights[row * P.w_row + (j0 + j) * P.w_col] : 1.f;
      const bool there = slot >= 0 && slot < total;
      if (!there) w[j] = 0.f;
      if (there) v[j] = *reinterpret_cast<const Vec<T, V> *>(rows + slot * P.y_stride + c);
      else v[j] = Vec<T, V>{};
    }
#pragma unroll
    for (int j = 0; j < B; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(w[j], to_f32(v[j].v[e]), acc[e]);
  }
  store_f32<T, V>(static_cast<T *>(P.out) + row * P.channels + c, acc);
}

// drows[slot] = w dout[t], dweights[t][j] = <dout[t], rows[slot]> (40 013 x 256 bf16, k 2: 20 us = 5.0 TB/s): G lanes per row of `dout`, two of the row's experts at a
// time, so that their gathers are in flight together and `dout` is read once for both.
template <typename T, int V, int G>
__global__ void __launch_bounds__(256) combine_backward_kernel(const MoveParams P) {
  pdl_trigger();
  pdl_wait();
  if (P.clear_here) clear_here<T, V>(P);
  const int g = threadIdx.x & (G - 1);
  const int vecs = P.channels / V;
  constexpr int kRows = 256 / G;
  const int64_t total = P.n * P.k, groups = (P.n + kRows - 1) / kRows;
  const T *dout = static_cast<const T *>(P.x), *rows = static_cast<const T *>(P.y);
  T *drows = static_cast<T *>(P.out);
  for (int64_t b = blockIdx.x; b < groups; b += gridDim.x) {
    const int64_t row = b * kRows + threadIdx.x / G;
    const bool live = row < P.n;
    for (int j0 = 0; j0 < P.k; j0 += 2) {
      int64_t slot[2];
      float w[2], dot[2] = {0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        slot[q] = live && j0 + q < P.k ? P.slots[row * P.k + j0 + q] : -1;
        if (slot[q] >= total) slot[q] = -1;
        w[q] = live && j0 + q < P.k && P.weights ? P.weights[row * P.w_row + (j0 + q) * P.w_col] : 1.f;
      }
      if (slot[0] >= 0 || slot[1] >= 0)
        for (int i = g; i < vecs; i += G) {
          float d[V], y[2][V];
          load_f32<T, V>(dout + row * P.x_stride + i * V, d);
          if (P.dweights)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (slot[q] >= 0) load_f32<T, V>(rows + slot[q] * P.y_stride + i * V, y[q]);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (slot[q] < 0) continue;
            if (P.dweights)
#pragma unroll
              for (int e = 0; e < V; ++e) dot[q] = fmaf(d[e], y[q][e], dot[q]);
            if (drows) {
              float o[V];
#pragma unroll
              for (int e = 0; e < V; ++e) o[e] = d[e] * w[q];
              store_f32<T, V>(drows + slot[q] * P.channels + i * V, o);
            }
          }
        }
      if (P.dweights) {
#pragma unroll
        for (int d = 1; d < G; d *= 2)
#pragma unroll
          for (int q = 0; q < 2; ++q) dot[q] += __shfl_xor_sync(0xffffffffu, dot[q], d, G);
        if (live && g < 2 && j0 + g < P.k) P.dweights[row * P.k + j0 + g] = g == 0 ? dot[0] : dot[1];
      }
    }
  }
  if (drows && P.offsets) zero_tail<T, V>(P, drows, vecs);
}

static std::atomic<int64_t> g_operator_launches{0};
void count_operator_launch() { g_operator_launches.fetch_add(1, std::memory_order_relaxed); }

static unsigned capped_blocks(int64_t work, int per_cta, int ctas_per_sm) {
  const int64_t want = div_up(work, per_cta), cap = static_cast<int64_t>(sm_count()) * ctas_per_sm;
  return static_cast<unsigned>(want < 1 ? 1 : want < cap ? want : cap);
}

// One CTA per SM, whole groups of 64 rows.
static int route_rows_per_cta(int64_t n, int64_t *rows_per_cta) {
  *rows_per_cta = div_up(div_up(n, sm_count()), 64) * 64;
  return static_cast<int>(div_up(n, *rows_per_cta));
}

static size_t stash_bytes(int lanes, int k) { return static_cast<size_t>(kRouteThreads / lanes) * k * 8; }
static size_t place_smem(int experts) { return static_cast<size_t>(3 * experts + 1 + kRouteWarps * (experts | 1)) * 4; }

// `most`: what the largest call of this kernel takes (many experts or a large k: up to 200 KB)
template <typename... KArgs>
static int launch_route_kernel(void (*kernel)(KArgs...), int ctas, size_t smem, size_t most, cudaStream_t st, const RouteParams &P) {
  const int rc = allow_smem(kernel, most);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_CUDA(launch_operator(kernel, dim3(ctas), dim3(kRouteThreads), smem, st, P));
  return SPIRA_B200_OK;
}

template <typename T, int G, int EPL>
static int launch_route(RouteParams &P, cudaStream_t st) {
  constexpr int kE = G * EPL, kK = kE < kMaxTopK ? kE : kMaxTopK;      // most experts and choices of this kernel
  auto small = [](int experts, int k) { return place_smem(experts) + stash_bytes(G, k); };
  auto choose = [](int experts, int k) { return static_cast<size_t>(experts) * 4 + stash_bytes(G, k); };
  if (P.n * P.k <= kSmallRouteEntries) return launch_route_kernel(route_small_kernel<T, G, EPL>, 1, small(P.experts, P.k), small(kE, kK), st, P);
  const int ctas = route_rows_per_cta(P.n, &P.rows_per_cta);
  const int rc = launch_route_kernel(route_choose_kernel<T, G, EPL>, ctas, choose(P.experts, P.k), choose(kE, kK), st, P);
  return rc != SPIRA_B200_OK ? rc : launch_route_kernel(route_place_kernel, ctas, place_smem(P.experts), place_smem(kMaxExperts), st, P);
}

template <typename T>
static int launch_route_lanes(RouteParams &P, cudaStream_t st) {
  // 16-bit logits of many rows: 32 experts per lane halve what every lane of a row does for itself (127 363 x 64: 19.7
  // instead of 23.2 us); with fewer rows half of the lanes would have none (20 000 x 64: 12.8 instead of 10.8 us)
  if (sizeof(T) == 2 && P.experts > 16 && P.n >= 400 * static_cast<int64_t>(sm_count())) {
    if (P.experts <= 32) return launch_route<T, 2, 16>(P, st);
    if (P.experts <= 64) return launch_route<T, 2, 32>(P, st);
    if (P.experts <= 128) return launch_route<T, 4, 32>(P, st);
    if (P.experts <= 256) return launch_route<T, 8, 32>(P, st);
    return launch_route<T, 16, 32>(P, st);
  }
  if (P.experts <= 8) return launch_route<T, 2, 4>(P, st);
  if (P.experts <= 16) return launch_route<T, 2, 8>(P, st);
  if (P.experts <= 32) return launch_route<T, 4, 8>(P, st);
  if (P.experts <= 64) return launch_route<T, 4, 16>(P, st);
  if (P.experts <= 128) return launch_route<T, 8, 16>(P, st);
  if (P.experts <= 256) return launch_route<T, 16, 16>(P, st);
  return launch_route<T, 32, 16>(P, st);
}

static int check_route(const char *what, int dtype, int64_t n, int64_t row_stride, int experts, int k) {
  SB_CHECK_ARG(dtype >= SPIRA_B200_F16 && dtype <= SPIRA_B200_F32, "%s: unknown element type %d", what, dtype);
  SB_CHECK_ARG(experts >= 1 && experts <= kMaxExperts, "%s: experts=%d must be 1 to %d", what, experts, kMaxExperts);
  SB_CHECK_ARG(k >= 1 && k <= kMaxTopK && k <= experts, "%s: top_k=%d must be 1 to min(experts, %d)", what, k, kMaxTopK);
  SB_CHECK_ARG(n >= 0 && n * k < (int64_t(1) << 31), "%s: %lld rows x %d experts are out of range", what, (long long)n, k);
  SB_CHECK_ARG(row_stride >= experts || n <= 1, "%s: row stride %lld is smaller than experts=%d", what, (long long)row_stride, experts);
  return SPIRA_B200_OK;
}

static int check_move(const char *what, const MoveParams &P, int dtype, int64_t stride_a, int64_t stride_b) {
  SB_CHECK_ARG(dtype >= SPIRA_B200_F16 && dtype <= SPIRA_B200_F32, "%s: unknown element type %d", what, dtype);
  SB_CHECK_ARG(P.k >= 1 && P.k <= kMaxTopK, "%s: top_k=%d must be 1 to %d", what, P.k, kMaxTopK);
  SB_CHECK_ARG(P.n >= 0 && P.n * P.k < (int64_t(1) << 31), "%s: %lld rows x %d experts are out of range", what, (long long)P.n, P.k);
  SB_CHECK_ARG(P.channels >= 1 && P.channels <= (1 << 20), "%s: channels=%d out of range", what, P.channels);
  SB_CHECK_ARG(stride_a >= 0 && stride_b >= 0, "%s: negative row stride", what);
  return SPIRA_B200_OK;
}

// 16-byte accesses need every row of every tensor to start on a 16-byte boundary.
static bool rows_aligned(const void *p, int64_t stride, int size) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0);
}

// For `ctas` CTAs that write the rows: by that one CTA, or by a launch before them.
static int launch_clear(MoveParams &P, int64_t ctas, int size, cudaStream_t st) {
  if (!P.clear || !P.out) return SPIRA_B200_OK;
  if (ctas == 1) {
    P.clear_here = 1;
    return SPIRA_B200_OK;
  }
  const int64_t total = P.n * P.k, row_bytes = static_cast<int64_t>(P.channels) * size;
  const dim3 grid(static_cast<unsigned>(div_up(total, 256)));
  unsigned char *rows = static_cast<unsigned char *>(P.out);
  if (rows_aligned(rows, P.channels, size)) SB_CHECK_CUDA(launch_operator(clear_kernel<16>, grid, dim3(256), 0, st, P.slots, P.order, total, row_bytes, rows));
  else if (size == 4) SB_CHECK_CUDA(launch_operator(clear_kernel<4>, grid, dim3(256), 0, st, P.slots, P.order, total, row_bytes, rows));
  else SB_CHECK_CUDA(launch_operator(clear_kernel<2>, grid, dim3(256), 0, st, P.slots, P.order, total, row_bytes, rows));
  return SPIRA_B200_OK;
}

template <typename T, int V>
static int launch_move(MoveParams &P, bool combine, cudaStream_t st) {
  const int64_t pieces = P.channels / V;
  P.rows_per_launch_row = ((int64_t(1) << 31) - 512) / pieces;
  if (P.rows_per_launch_row > P.n) P.rows_per_launch_row = P.n;
  int bits = 0;
  while ((int64_t(1) << bits) < pieces) ++bits;
  P.div_shift = 31 + bits;
  P.div_mul = ((uint64_t(1) << P.div_shift) + pieces - 1) / pieces;
  const dim3 grid(static_cast<unsigned>(div_up(P.rows_per_launch_row * pieces, 256)), static_cast<unsigned>(div_up(P.n, P.rows_per_launch_row)));
  SB_CHECK_ARG(grid.y < 65536, "too many rows x channels");
  if (!combine) {
    const int rc = launch_clear(P, static_cast<int64_t>(grid.x) * grid.y, sizeof(T), st);
    if (rc != SPIRA_B200_OK) return rc;
  }
  auto go = [&](auto kernel) -> int {
    SB_CHECK_CUDA(launch_operator(kernel, grid, dim3(256), 0, st, P));
    return SPIRA_B200_OK;
  };
  if (combine) return P.k == 1 ? go(combine_kernel<T, V, 1>) : P.k == 2 ? go(combine_kernel<T, V, 2>) : P.k == 4 ? go(combine_kernel<T, V, 4>) : go(combine_kernel<T, V, 0>);
  return P.k == 1 ? go(dispatch_kernel<T, V, 1>) : P.k == 2 ? go(dispatch_kernel<T, V, 2>) : P.k == 4 ? go(dispatch_kernel<T, V, 4>) : go(dispatch_kernel<T, V, 0>);
}

template <typename T, int V>
static int launch_combine_backward(MoveParams &P, cudaStream_t st) {
  const int vecs = P.channels / V;
  // as many lanes as the row has pieces, half of them where the rows fill the SMs all the same: two pieces per lane are in
  // flight together (127 363 x 96, k 2: 28 instead of 33 us; 20 000 x 64, k 8: 13 with all lanes, 20 us with half).  No
  // more CTAs than fit at once (39 us).
  int lanes = vecs <= 4 ? 4 : vecs <= 8 ? 8 : vecs <= 16 ? 16 : 32;
  if (lanes > 4 && vecs <= 32 && P.n * (lanes / 2) >= 4 * 256 * static_cast<int64_t>(sm_count())) lanes /= 2;
  const unsigned blocks = capped_blocks(P.n * lanes, 256, 8);
  const int rc = launch_clear(P, blocks, sizeof(T), st);
  if (rc != SPIRA_B200_OK) return rc;
  if (lanes == 4) SB_CHECK_CUDA(launch_operator(combine_backward_kernel<T, V, 4>, dim3(blocks), dim3(256), 0, st, P));
  else if (lanes == 8) SB_CHECK_CUDA(launch_operator(combine_backward_kernel<T, V, 8>, dim3(blocks), dim3(256), 0, st, P));
  else if (lanes == 16) SB_CHECK_CUDA(launch_operator(combine_backward_kernel<T, V, 16>, dim3(blocks), dim3(256), 0, st, P));
  else SB_CHECK_CUDA(launch_operator(combine_backward_kernel<T, V, 32>, dim3(blocks), dim3(256), 0, st, P));
  return SPIRA_B200_OK;
}

static int run_dispatch(MoveParams &P, int dtype, cudaStream_t st) {
  const int size = elem_size(dtype);
  const bool wide = P.channels * size % 16 == 0 && rows_aligned(P.x, P.x_stride, size) && rows_aligned(P.out, P.channels, size);
  return SB_DISPATCH_ELEM(dtype, T, {
    if (wide) return launch_move<T, 16 / static_cast<int>(sizeof(T))>(P, false, st);
    return launch_move<T, 1>(P, false, st);
  });
}

static int run_combine_backward(MoveParams &P, int dtype, cudaStream_t st) {
  const int size = elem_size(dtype);
  const bool wide = P.channels * size % 16 == 0 && rows_aligned(P.y, P.y_stride, size) && rows_aligned(P.x, P.x_stride, size) &&
                    rows_aligned(P.out, P.channels, size);
  return SB_DISPATCH_ELEM(dtype, T, {
    if (wide) return launch_combine_backward<T, 16 / static_cast<int>(sizeof(T))>(P, st);
    return launch_combine_backward<T, 1>(P, st);
  });
}

}  // namespace sb

using namespace sb;

extern "C" int spira_b200_operator_launches(int64_t *count) {
  SB_CHECK_ARG(count, "operator_launches: null pointer");
  *count = g_operator_launches.load(std::memory_order_relaxed);
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_expert_route_workspace(int64_t n, int experts, int k, size_t *bytes) {
  int rc = check_route("expert_route", SPIRA_B200_F32, n, experts, experts, k);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(bytes, "expert_route: null pointer");
  int64_t rows;
  *bytes = n * k <= kSmallRouteEntries ? 0 : static_cast<size_t>(route_rows_per_cta(n, &rows)) * experts * 4;
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_expert_route(const void *logits, int dtype, int64_t n, int64_t row_stride, int experts, int k, int renormalize,
                                       float *weights, int32_t *chosen, int32_t *slots, int32_t *order, int32_t *offsets, void *workspace,
                                       size_t workspace_bytes, void *stream) {
  int rc = check_route("expert_route", dtype, n, row_stride, experts, k);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(offsets && (n == 0 || (logits && weights && chosen && slots && order)), "expert_route: null pointer");
  size_t need = 0;
  rc = spira_b200_expert_route_workspace(n, experts, k, &need);
  if (rc != SPIRA_B200_OK) return rc;
  if (workspace_bytes < need || (need && !workspace))
    return fail(SPIRA_B200_ERR_WORKSPACE, "expert_route: workspace of %zu bytes is smaller than %zu", workspace_bytes, need);
  RouteParams P{logits, n, row_stride, 0, experts, k, renormalize != 0, weights, chosen, slots, order, offsets, static_cast<int *>(workspace)};
  return SB_DISPATCH_ELEM(dtype, T, return launch_route_lanes<T>(P, as_stream(stream)););
}

extern "C" int spira_b200_expert_route_backward(const void *logits, int dtype, int64_t n, int64_t row_stride, int experts, int k,
                                                int renormalize, const float *weights, const int32_t *chosen, const float *dweights,
                                                int64_t dweights_row, int64_t dweights_col, void *dlogits, void *stream) {
  int rc = check_route("expert_route_backward", dtype, n, row_stride, experts, k);
  if (rc != SPIRA_B200_OK || n == 0) return rc;
  SB_CHECK_ARG(logits && weights && chosen && dweights && dlogits, "expert_route_backward: null pointer");
  cudaStream_t st = as_stream(stream);
  return SB_DISPATCH_ELEM(dtype, T, {
    const T *l = static_cast<const T *>(logits);
    T *d = static_cast<T *>(dlogits);
    auto go = [&](auto kernel, int lanes) -> int {
      SB_CHECK_CUDA(launch_operator(kernel, dim3(static_cast<unsigned>(div_up(n * lanes, 256))), dim3(256), 0, st, l, n, row_stride, experts, k,
                                     renormalize != 0 ? 1 : 0, weights, chosen, dweights, dweights_row, dweights_col, d));
      return SPIRA_B200_OK;
    };
    if (experts <= 8) return go(route_backward_kernel<T, 2, 4>, 2);
    if (experts <= 16) return go(route_backward_kernel<T, 4, 4>, 4);
    if (experts <= 32) return go(route_backward_kernel<T, 8, 4>, 8);
    if (experts <= 64) return go(route_backward_kernel<T, 16, 4>, 16);
    if (experts <= 128) return go(route_backward_kernel<T, 32, 4>, 32);
    return go(route_backward_kernel<T, 32, 16>, 32);
  });
}

extern "C" int spira_b200_expert_dispatch(const void *x, int dtype, int64_t n, int64_t x_stride, int channels, const int32_t *slots, int k,
                                          const int32_t *offsets, int experts, void *rows, void *stream) {
  MoveParams P{};
  P.x = x; P.slots = slots; P.offsets = offsets; P.out = rows;
  P.n = n; P.x_stride = x_stride; P.channels = channels; P.k = k; P.experts = experts;
  int rc = check_move("expert_dispatch", P, dtype, x_stride, 0);
  if (rc != SPIRA_B200_OK || n == 0) return rc;
  SB_CHECK_ARG(x && slots && offsets && rows && experts >= 1, "expert_dispatch: null pointer");
  return run_dispatch(P, dtype, as_stream(stream));
}

extern "C" int spira_b200_expert_dispatch_cleared(const void *x, int dtype, int64_t n, int64_t x_stride, int channels, const int32_t *slots,
                                                  const int32_t *order, int k, void *rows, void *stream) {
  MoveParams P{};
  P.x = x; P.slots = slots; P.order = order; P.out = rows; P.clear = 1;
  P.n = n; P.x_stride = x_stride; P.channels = channels; P.k = k;
  int rc = check_move("expert_dispatch_cleared", P, dtype, x_stride, 0);
  if (rc != SPIRA_B200_OK || n == 0) return rc;
  SB_CHECK_ARG(x && slots && rows, "expert_dispatch_cleared: null pointer");
  return run_dispatch(P, dtype, as_stream(stream));
}

extern "C" int spira_b200_expert_combine(const void *rows, int dtype, int64_t n, int64_t row_stride, int channels, const float *weights,
                                         int64_t weights_row, int64_t weights_col, const int32_t *slots, int k, void *out, void *stream) {
  MoveParams P{};
  P.y = rows; P.weights = weights; P.slots = slots; P.out = out; P.w_row = weights_row; P.w_col = weights_col;
  P.n = n; P.y_stride = row_stride; P.channels = channels; P.k = k;
  int rc = check_move("expert_combine", P, dtype, row_stride, 0);
  if (rc != SPIRA_B200_OK || n == 0) return rc;
  SB_CHECK_ARG(rows && slots && out, "expert_combine: null pointer");
  const int size = elem_size(dtype);
  const bool wide = channels * size % 16 == 0 && rows_aligned(rows, row_stride, size) && rows_aligned(out, channels, size);
  cudaStream_t st = as_stream(stream);
  return SB_DISPATCH_ELEM(dtype, T, {
    if (wide) return launch_move<T, 16 / static_cast<int>(sizeof(T))>(P, true, st);
    return launch_move<T, 1>(P, true, st);
  });
}

extern "C" int spira_b200_expert_combine_backward(const void *rows, const void *dout, int dtype, int64_t n, int64_t row_stride, int64_t dout_stride,
                                                  int channels, const float *weights, int64_t weights_row, int64_t weights_col,
                                                  const int32_t *slots, int k, const int32_t *offsets, int experts, void *drows,
                                                  float *dweights, void *stream) {
  MoveParams P{};
  P.x = dout; P.y = rows; P.weights = weights; P.slots = slots; P.offsets = offsets; P.out = drows; P.dweights = dweights;
  P.n = n; P.x_stride = dout_stride; P.y_stride = row_stride; P.w_row = weights_row; P.w_col = weights_col;
  P.channels = channels; P.k = k; P.experts = experts;
  int rc = check_move("expert_combine_backward", P, dtype, row_stride, dout_stride);
  if (rc != SPIRA_B200_OK || n == 0) return rc;
  SB_CHECK_ARG(dout && slots && offsets && experts >= 1 && (rows || !dweights) && (drows || dweights), "expert_combine_backward: null pointer");
  return run_combine_backward(P, dtype, as_stream(stream));
}

extern "C" int spira_b200_expert_combine_backward_cleared(const void *rows, const void *dout, int dtype, int64_t n, int64_t row_stride,
                                                          int64_t dout_stride, int channels, const float *weights, int64_t weights_row,
                                                          int64_t weights_col, const int32_t *slots, const int32_t *order, int k, void *drows,
                                                          float *dweights, void *stream) {
  MoveParams P{};
  P.x = dout; P.y = rows; P.weights = weights; P.slots = slots; P.order = order; P.out = drows; P.dweights = dweights; P.clear = 1;
  P.n = n; P.x_stride = dout_stride; P.y_stride = row_stride; P.w_row = weights_row; P.w_col = weights_col;
  P.channels = channels; P.k = k;
  int rc = check_move("expert_combine_backward_cleared", P, dtype, row_stride, dout_stride);
  if (rc != SPIRA_B200_OK || n == 0) return rc;
  SB_CHECK_ARG(dout && slots && (rows || !dweights) && (drows || dweights), "expert_combine_backward_cleared: null pointer");
  return run_combine_backward(P, dtype, as_stream(stream));
}
