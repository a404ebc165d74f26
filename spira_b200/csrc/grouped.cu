// Ragged products of grouped rows with one weight matrix per group (the experts of a mixture):
//
//   y[r]  = relu?(x[r] W[e] + b[e])      rows r of group e
//   dz    = dy (y > 0)                    db[e] = sum over the group's rows of dz
//   dx[r] = dz[r] W[e]^T                  dW[e] = x_e^T dz_e
//
// Rows outside every group are zero in y and dx.  Group boundaries are read on the device; the host only knows upper
// bounds of the tile counts.  Sums over a group's rows are split into pieces that are added in a fixed order.
//
// Channel counts in whole 16-byte units and aligned tensors run on the tensor-core kernel (grouped_tc.cu).
// `grouped_any_kernel` takes every channel count, stride and alignment: 64 x 64 tiles, element-wise loads into shared
// memory, warp-level MMAs with fp32 accumulation.
#include "common.cuh"
#include "elem.cuh"
#include "grouped.cuh"

namespace sb {

static_assert(sizeof(spira_b200_grouped_desc) == 128, "spira_b200_grouped_desc layout");

constexpr int kATile = 64, kAK = 32, kALd = kAK + 8;     // (row stride of 80 bytes: conflict-free fragment loads)
constexpr int kAThreads = 128;

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct GroupedParams {
  const void *a, *b, *bias;       // forward: x, W; dx: dz, W; dW: x, dz
  const int32_t *offsets;
  void *out;
  float *partial;                 // dW with several pieces per group: [pieces][c_in][c_out]
  int64_t a_stride, b_stride;
  int n, experts, c_in, c_out, relu, piece;
};

template <typename T>
__device__ __forceinline__ void zero_outside(T *out, int channels, int n, const int32_t *offsets, int experts) {
  int first, last;
  group_span(offsets, experts, n, first, last);
  const int64_t threads = static_cast<int64_t>(gridDim.x) * gridDim.y * blockDim.x;
  const int64_t me = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = me; i < static_cast<int64_t>(first) * channels; i += threads) out[i] = from_f32<T>(0.f);
  for (int64_t i = static_cast<int64_t>(last) * channels + me; i < static_cast<int64_t>(n) * channels; i += threads) out[i] = from_f32<T>(0.f);
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kAThreads) grouped_any_kernel(const __grid_constant__ GroupedParams P) {
  __shared__ __align__(16) T sa[kATile * kALd], sb_[kATile * kALd];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (MODE != kDw) zero_outside(static_cast<T *>(P.out), MODE == kForward ? P.c_out : P.c_in, P.n, P.offsets, P.experts);
  int expert, m0, n0, m_end, n_end, k_begin, k_end;
  int64_t unit = 0;
  if (MODE == kDw) {
    // one piece of one group's rows, one tile of the weight matrix (piece == 0: the whole group)
    if (P.piece == 0) {
      expert = blockIdx.x;
      int lo = clamped_offset(P.offsets, 0, P.n), hi = lo;
      for (int e = 1; e <= expert + 1; ++e) {
        if (e == expert + 1) lo = hi;
        const int v = clamped_offset(P.offsets, e, P.n);
        hi = v > hi ? v : hi;
      }
      k_begin = lo;
      k_end = hi;
    } else {
      const GroupTile t = find_group_tile(P.offsets, P.experts, P.n, P.piece, blockIdx.x);
      if (t.expert < 0) return;
      expert = t.expert;
      unit = blockIdx.x;
      k_begin = t.begin + t.index * P.piece;
      k_end = k_begin + P.piece < t.end ? k_begin + P.piece : t.end;
    }
    const int m_tiles = (P.c_in + kATile - 1) / kATile;
    m0 = static_cast<int>(blockIdx.y) % m_tiles * kATile;
    n0 = static_cast<int>(blockIdx.y) / m_tiles * kATile;
    m_end = P.c_in;
    n_end = P.c_out;
  } else {
    const GroupTile t = find_group_tile(P.offsets, P.experts, P.n, kATile, blockIdx.x);
    if (t.expert < 0) return;
    expert = t.expert;
    m0 = t.begin + t.index * kATile;
    m_end = t.end;
    n0 = blockIdx.y * kATile;
    n_end = MODE == kForward ? P.c_out : P.c_in;
    k_begin = 0;
    k_end = MODE == kForward ? P.c_in : P.c_out;
  }
  const T zero = from_f32<T>(0.f);
  const T *A = static_cast<const T *>(P.a);
  const T *B = static_cast<const T *>(P.b);
  if (MODE != kDw) B += static_cast<int64_t>(expert) * P.c_in * P.c_out;
  const int g = lane >> 2, t4 = lane & 3;
  const int wm = (warp & 1) * 32, wn = (warp >> 1) * 32;
  float acc[2][4][4] = {};
  // neighbouring threads follow the direction in which the source is contiguous; the next step's elements are on their way
  // while this step multiplies
  constexpr int kEach = kATile * kAK / kAThreads;
  T ra[kEach], rb[kEach];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const int i = tid + q * kAThreads;
      const int m = MODE == kDw ? i % kATile : i / kAK, k = MODE == kDw ? i / kATile : i % kAK;
      ra[q] = zero;
      if (m0 + m < m_end && k0 + k < k_end)
        ra[q] = MODE == kDw ? A[static_cast<int64_t>(k0 + k) * P.a_stride + m0 + m] : A[static_cast<int64_t>(m0 + m) * P.a_stride + k0 + k];
    }
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const int i = tid + q * kAThreads;
      const int n = MODE == kDx ? i / kAK : i % kATile, k = MODE == kDx ? i % kAK : i / kATile;
      rb[q] = zero;
      if (n0 + n < n_end && k0 + k < k_end) {
        if (MODE == kForward) rb[q] = B[static_cast<int64_t>(k0 + k) * P.c_out + n0 + n];
        else if (MODE == kDx) rb[q] = B[static_cast<int64_t>(n0 + n) * P.c_out + k0 + k];
        else rb[q] = B[static_cast<int64_t>(k0 + k) * P.b_stride + n0 + n];
      }
    }
  };
  fetch(k_begin);
  for (int k0 = k_begin; k0 < k_end; k0 += kAK) {
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const int i = tid + q * kAThreads;
      const int m = MODE == kDw ? i % kATile : i / kAK, ka = MODE == kDw ? i / kATile : i % kAK;
      const int n = MODE == kDx ? i / kAK : i % kATile, kb = MODE == kDx ? i % kAK : i / kATile;
      sa[m * kALd + ka] = ra[q];
      sb_[n * kALd + kb] = rb[q];
    }
    fetch(k0 + kAK);
    __syncthreads();
    const uint32_t *a32 = reinterpret_cast<const uint32_t *>(sa), *b32 = reinterpret_cast<const uint32_t *>(sb_);
#pragma unroll
    for (int ks = 0; ks < kAK / 16; ++ks) {
      uint32_t a[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t *p = a32 + (wm + 16 * i + g) * (kALd / 2) + ks * 8 + t4;
        a[i][0] = p[0];
        a[i][1] = p[8 * (kALd / 2)];
        a[i][2] = p[4];
        a[i][3] = p[8 * (kALd / 2) + 4];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t *p = b32 + (wn + 8 * j + g) * (kALd / 2) + ks * 8 + t4;
        const uint32_t b0 = p[0], b1 = p[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) mma_16816<T>(acc[i][j], a[i], b0, b1);
      }
    }
    __syncthreads();
  }
  T *out = static_cast<T *>(P.out);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = m0 + wm + 16 * i + g + 8 * (q >> 1), n = n0 + wn + 8 * j + 2 * t4 + (q & 1);
        if (m >= m_end || n >= n_end) continue;
        float v = acc[i][j][q];
        if (MODE == kForward) {
          if (P.bias) v += to_f32(static_cast<const T *>(P.bias)[static_cast<int64_t>(expert) * P.c_out + n]);
          if (P.relu) v = v < 0.f ? 0.f : v;          // (a NaN stays)
          out[static_cast<int64_t>(m) * P.c_out + n] = from_f32<T>(v);
        } else if (MODE == kDx) {
          out[static_cast<int64_t>(m) * P.c_in + n] = from_f32<T>(v);
        } else if (P.piece == 0) {
          out[(static_cast<int64_t>(expert) * P.c_in + m) * P.c_out + n] = from_f32<T>(v);
        } else {
          P.partial[(unit * P.c_in + m) * P.c_out + n] = v;
        }
      }
}

// Number of the first piece of group e and how many it has, by every warp for itself.
__device__ __forceinline__ void group_pieces(const int32_t *offsets, int n, int e, int piece, int64_t &first, int &count) {
  const int lane = threadIdx.x & 31;
  int before = 0, highest = 0, last = 0;
  for (int i0 = 0; i0 <= e; i0 += 32) {
    const int i = i0 + lane;
    int lo = i <= e ? clamped_offset(offsets, i, n) : 0;
    int hi = i <= e ? clamped_offset(offsets, i + 1, n) : 0;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, lo, d);
      if (lane >= d && o > lo) lo = o;
    }
    lo = lo > highest ? lo : highest;
    hi = hi > lo ? hi : lo;
    const int mine = i <= e ? (hi - lo + piece - 1) / piece : 0;
    int sum = mine;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    before += sum;
    const int src = e - i0 < 31 ? e - i0 : 31;
    last = __shfl_sync(0xffffffffu, mine, src);
    highest = __shfl_sync(0xffffffffu, hi, 31);
  }
  first = before - last;
  count = last;
}

// out[e][i] = sum over the pieces of group e, in order, of partial[piece][i]
template <typename T>
__global__ void __launch_bounds__(256) grouped_sum_kernel(const float *partial, const int32_t *offsets, int n, int experts, int piece, int64_t size, T *out) {
  pdl_trigger();
  pdl_wait();
  const int e = blockIdx.y;
  int64_t first;
  int count;
  group_pieces(offsets, n, e, piece, first, count);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < size; i += static_cast<int64_t>(gridDim.x) * 256) {
    float t = 0.f;
#pragma unroll 4
    for (int p = 0; p < count; ++p) t += partial[(first + p) * size + i];
    out[e * size + i] = from_f32<T>(t);
  }
}

// dz = dy where the ReLU let the value through (dz != NULL), and column sums over pieces of a group's rows.  What the ReLU
// let through: MASK 1 a bit per element that the forward pass wrote, 2 y > 0, 0 everything (no ReLU).  A copy with four
// rows of a thread in flight; four CTAs per SM.
template <typename T, int V, int MASK>
__global__ void __launch_bounds__(256, 4) grouped_dz_kernel(const T *dy, int64_t dy_stride, const T *y, const unsigned char *mask, int mask_pitch, T *dz,
                                                            float *partial, const int32_t *offsets, int n, int experts, int c_out, int piece) {
  __shared__ float sums[256 * V];
  pdl_trigger();
  pdl_wait();
  const GroupTile t = find_group_tile(offsets, experts, n, piece, blockIdx.x);
  if (t.expert < 0) return;
  const int r0 = t.begin + t.index * piece, r1 = r0 + piece < t.end ? r0 + piece : t.end;
  const int vecs = c_out / V, wide = vecs - static_cast<int>(blockIdx.y) * 256 < 256 ? vecs - static_cast<int>(blockIdx.y) * 256 : 256;
  const int lanes = 256 / wide;                 // rows in parallel
  const int lane = threadIdx.x / wide, c = (blockIdx.y * 256 + threadIdx.x % wide) * V;
  constexpr int kBatch = 4;                     // rows of a thread in flight
  float sum[V] = {};
  if (lane < lanes)
    for (int r = r0 + lane; r < r1; r += kBatch * lanes) {
      Vec<T, V> d[kBatch], f[MASK == 2 ? kBatch : 1];
      unsigned bits[MASK == 1 ? kBatch : 1];
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int row = r + q * lanes < r1 ? r + q * lanes : r;      // (past the end: the first row again, not used)
        d[q] = *reinterpret_cast<const Vec<T, V> *>(dy + row * dy_stride + c);
        if (MASK == 1) bits[q] = mask[static_cast<int64_t>(row) * mask_pitch + c / 8] >> (c & 7);
        if (MASK == 2) f[q] = *reinterpret_cast<const Vec<T, V> *>(y + static_cast<int64_t>(row) * c_out + c);
      }
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int64_t row = r + q * lanes;
        if (row >= r1) break;
        if (MASK == 1 && V == 8) {
          uint32_t *w = reinterpret_cast<uint32_t *>(&d[q]);
#pragma unroll
          for (int i = 0; i < V / 2; ++i) w[i] &= (bits[q] >> 2 * i & 1u) * 0xffffu | (bits[q] >> (2 * i + 1) & 1u) * 0xffff0000u;
        } else if (MASK != 0) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (MASK == 1 ? !(bits[q] >> i & 1) : !(to_f32(f[q].v[i]) > 0.f)) d[q].v[i] = from_f32<T>(0.f);
        }
        if (dz) *reinterpret_cast<Vec<T, V> *>(dz + row * c_out + c) = d[q];
        float v[V];
        vec_to_f32<T, V>(d[q], v);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += v[i];
      }
    }
  if (partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < V; ++i) sums[threadIdx.x * V + i] = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < wide * V; i += 256) {
    float s = 0.f;
    for (int l = 0; l < lanes; ++l) s += sums[(l * wide) * V + i];
    partial[static_cast<int64_t>(blockIdx.x) * c_out + blockIdx.y * 256 * V + i] = s;
  }
}

// Column sums of many short pieces: 32 columns x 32 strides of pieces per block, then a fixed tree.
template <typename T>
__global__ void __launch_bounds__(1024) grouped_column_sum_kernel(const float *partial, const int32_t *offsets, int n, int experts, int piece, int size, T *out) {
  __shared__ float part[32][33];
  pdl_trigger();
  pdl_wait();
  const int e = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  int64_t first;
  int count;
  group_pieces(offsets, n, e, piece, first, count);
  float t = 0.f;
  if (c < size)
#pragma unroll 4
    for (int p = w; p < count; p += 32) t += partial[(first + p) * size + c];
  part[w][lane] = t;
  __syncthreads();
  t = part[lane][w];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) t += __shfl_xor_sync(0xffffffffu, t, d);
  const int co = blockIdx.x * 32 + w;
  if (lane == 0 && co < size) out[static_cast<int64_t>(e) * size + co] = from_f32<T>(t);
}

// Rows per piece of the column sums: a CTA per piece, all of them resident at once (four per SM), at least 32 rows.
static int dz_piece(int64_t n) {
  const int64_t p = div_up(div_up(n, 15 * sm_count() / 4), 8) * 8;
  return static_cast<int>(p < 32 ? 32 : p);
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of a group that one CTA of the weight gradient adds up (0: all of them).  Splitting fills the SMs when the weight
// matrices have few tiles, at the price of fp32 partial sums: `ctas` per SM, at least 128 rows each.
static int dw_piece(int64_t n, int experts, int64_t tiles, int ctas) {
  if (tiles * experts >= sm_count() || n <= 128) return 0;
  const int64_t pieces = div_up(ctas * static_cast<int64_t>(sm_count()), tiles);
  int64_t piece = div_up(div_up(n, pieces), 64) * 64;
  if (piece < 128) piece = 128;
  return piece >= n ? 0 : static_cast<int>(piece);
}

// Which kernel a product runs on; one answer for a call and for its workspace.
static bool tc_forward(const spira_b200_grouped_desc &D) {
  return grouped_tc_available() && D.c_out % 8 == 0 && grouped_tc_rows_ok(D.x, D.x_stride, D.c_in, D.n) && aligned16(D.weight) && aligned16(D.bias) && aligned16(D.y);
}
static bool tc_dx(const spira_b200_grouped_desc &D) {
  return grouped_tc_available() && D.c_in % 8 == 0 && grouped_tc_rows_ok(D.dy, D.dy_stride, D.c_out, D.n) && aligned16(D.weight) && aligned16(D.dx);
}
static bool tc_dw(const spira_b200_grouped_desc &D) {
  return grouped_tc_available() && grouped_tc_rows_ok(D.x, D.x_stride, D.c_in, D.n) && grouped_tc_rows_ok(D.dy, D.dy_stride, D.c_out, D.n) && aligned16(D.dweight);
}
static unsigned long long wait_ns() { return static_cast<unsigned long long>(spira_b200_get_option("wait_limit_us")) * 1000ull; }

static int64_t any_tiles(int c_in, int c_out) { return div_up(c_in, kATile) * div_up(c_out, kATile); }

static int dw_rows(const spira_b200_grouped_desc &D) {
  return tc_dw(D) ? dw_piece(D.n, D.experts, grouped_tc_dw_tiles(D.c_in, D.c_out), 1) : dw_piece(D.n, D.experts, any_tiles(D.c_in, D.c_out), 2);
}

static int grouped_check(const char *what, const spira_b200_grouped_desc *D) {
  SB_CHECK_ARG(D, "%s: null descriptor", what);
  SB_CHECK_ARG(D->dtype == SPIRA_B200_F16 || D->dtype == SPIRA_B200_BF16, "%s: element type %d is neither fp16 nor bf16", what, D->dtype);
  SB_CHECK_ARG(D->n >= 0 && D->n < (int64_t(1) << 31) - 4096, "%s: n=%lld out of range", what, (long long)D->n);
  SB_CHECK_ARG(D->experts >= 1 && D->experts <= kMaxGroups, "%s: experts=%d must be 1 to %d", what, D->experts, kMaxGroups);
  SB_CHECK_ARG(D->c_in >= 1 && D->c_in <= 65536 && D->c_out >= 1 && D->c_out <= 65536, "%s: channels %d -> %d out of range", what, D->c_in, D->c_out);
  SB_CHECK_ARG(D->x_stride >= 0 && D->dy_stride >= 0, "%s: negative row stride", what);
  SB_CHECK_ARG(D->n == 0 || D->offsets, "%s: null pointer", what);
  return SPIRA_B200_OK;
}

template <typename T, int MODE>
static int launch_any(const GroupedParams &P, cudaStream_t st) {
  const int64_t units = MODE == kDw ? (P.piece ? group_tiles_bound(P.n, P.experts, P.piece) : P.experts) : group_tiles_bound(P.n, P.experts, kATile);
  const int64_t columns = MODE == kForward ? div_up(P.c_out, kATile) : MODE == kDx ? div_up(P.c_in, kATile) : any_tiles(P.c_in, P.c_out);
  SB_CHECK_ARG(columns < 65536 && units < (int64_t(1) << 31), "grouped_linear: too many tiles");
  SB_CHECK_CUDA(launch_dependent(grouped_any_kernel<T, MODE>, dim3(static_cast<unsigned>(units < 1 ? 1 : units), static_cast<unsigned>(columns)),
                                 dim3(kAThreads), 0, st, P));
  return SPIRA_B200_OK;
}

}  // namespace sb

using namespace sb;

#define SB_DISPATCH_HALF(dtype, T, ...)                              \
  [&]() -> int {                                                     \
    if ((dtype) == SPIRA_B200_F16) { using T = __half; __VA_ARGS__ } \
    using T = __nv_bfloat16; __VA_ARGS__                             \
  }()

extern "C" int spira_b200_grouped_linear(const spira_b200_grouped_desc *desc, int32_t *status, void *stream) {
  int rc = grouped_check("grouped_linear", desc);
  if (rc != SPIRA_B200_OK || desc->n == 0) return rc;
  const spira_b200_grouped_desc &D = *desc;
  SB_CHECK_ARG(D.x && D.weight && D.y, "grouped_linear: null pointer");
  SB_CHECK_ARG(!D.mask || (D.relu && tc_forward(D)), "grouped_linear: no mask is written for this call (spira_b200_grouped_linear_mask_bytes is 0)");
  if (tc_forward(D)) return grouped_tc_run(kForward, D, 0, nullptr, status, wait_ns(), as_stream(stream));
  GroupedParams P{D.x, D.weight, D.bias, D.offsets, D.y, nullptr, D.x_stride, 0, static_cast<int>(D.n), D.experts, D.c_in, D.c_out, D.relu, 0};
  return SB_DISPATCH_HALF(D.dtype, T, return (launch_any<T, kForward>(P, as_stream(stream))););
}

extern "C" int spira_b200_grouped_linear_mask_bytes(const spira_b200_grouped_desc *desc, size_t *bytes) {
  int rc = grouped_check("grouped_linear_mask", desc);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(bytes, "grouped_linear_mask: null pointer");
  *bytes = desc->n > 0 && desc->relu && tc_forward(*desc) ? static_cast<size_t>(desc->n) * mask_pitch(desc->c_out) : 0;
  return SPIRA_B200_OK;
}

// Scratch of the backward pass: dz where a ReLU followed, then the partial sums (of dbias, later of dweight: one region).
struct BackwardPlan {
  bool need_dz;
  int dz_rows, dw_rows;
  size_t partial_at, bytes;
};

static BackwardPlan backward_plan(const spira_b200_grouped_desc &D, const spira_b200_grouped_desc &Z) {
  BackwardPlan p{};
  p.need_dz = D.relu && (D.dx || D.dweight);
  p.dz_rows = dz_piece(D.n);
  p.dw_rows = D.dweight ? dw_rows(Z) : 0;
  p.partial_at = p.need_dz ? static_cast<size_t>(div_up(D.n * D.c_out * 2, 256) * 256) : 0;
  const size_t db = D.dbias ? static_cast<size_t>(group_tiles_bound(D.n, D.experts, p.dz_rows)) * D.c_out * 4 : 0;
  const size_t dw = p.dw_rows ? static_cast<size_t>(group_tiles_bound(D.n, D.experts, p.dw_rows)) * D.c_in * D.c_out * 4 : 0;
  p.bytes = p.partial_at + (db > dw ? db : dw);
  return p;
}

// The call with dz in the place of dy.
static spira_b200_grouped_desc with_dz(const spira_b200_grouped_desc &D, const void *workspace) {
  spira_b200_grouped_desc Z = D;
  if (D.relu && (D.dx || D.dweight)) {
    Z.dy = workspace;
    Z.dy_stride = D.c_out;
  }
  return Z;
}

static int backward_check(const spira_b200_grouped_desc *D) {
  int rc = grouped_check("grouped_linear_backward", D);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(D->dx || D->dweight || D->dbias || D->n == 0, "grouped_linear_backward: no gradient is asked for");
  SB_CHECK_ARG(D->n == 0 || (D->dy && (!D->dx || D->weight) && (!D->dweight || D->x) && (!D->relu || D->mask || D->y)),
               "grouped_linear_backward: null pointer");
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_grouped_linear_backward_workspace(const spira_b200_grouped_desc *desc, size_t *bytes) {
  int rc = backward_check(desc);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(bytes, "grouped_linear_backward: null pointer");
  *bytes = desc->n ? backward_plan(*desc, with_dz(*desc, nullptr)).bytes : 0;
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_grouped_linear_backward(const spira_b200_grouped_desc *desc, void *workspace, size_t workspace_bytes, int32_t *status,
                                                  void *stream) {
  int rc = backward_check(desc);
  if (rc != SPIRA_B200_OK) return rc;
  const spira_b200_grouped_desc &D = *desc;
  cudaStream_t st = as_stream(stream);
  const int64_t size = static_cast<int64_t>(D.c_in) * D.c_out;
  if (D.n == 0) {
    if (D.dweight) SB_CHECK_CUDA(cudaMemsetAsync(D.dweight, 0, static_cast<size_t>(D.experts) * size * 2, st));
    if (D.dbias) SB_CHECK_CUDA(cudaMemsetAsync(D.dbias, 0, static_cast<size_t>(D.experts) * D.c_out * 2, st));
    return SPIRA_B200_OK;
  }
  const spira_b200_grouped_desc Z = with_dz(D, workspace);
  const BackwardPlan plan = backward_plan(D, with_dz(D, nullptr));      // (as the size was asked for: dz is aligned like a null pointer)
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
    return fail(SPIRA_B200_ERR_WORKSPACE, "grouped_linear_backward: workspace of %zu bytes is smaller than %zu", workspace_bytes, plan.bytes);
  SB_CHECK_ARG(aligned16(workspace), "grouped_linear_backward: the workspace must be 16-byte aligned");
  float *partial = reinterpret_cast<float *>(static_cast<unsigned char *>(workspace) + plan.partial_at);
  const int n = static_cast<int>(D.n);
  return SB_DISPATCH_HALF(D.dtype, T, {
    if (plan.need_dz || D.dbias) {
      T *dz = plan.need_dz ? static_cast<T *>(workspace) : nullptr;
      const unsigned units = static_cast<unsigned>(group_tiles_bound(n, D.experts, plan.dz_rows));
      const bool wide = D.c_out % 8 == 0 && aligned16(D.dy) && (D.dy_stride % 8 == 0 || n == 1) && (D.mask || aligned16(D.y));
      auto go = [&](auto kernel, int columns) -> int {
        SB_CHECK_CUDA(launch_dependent(kernel, dim3(units, static_cast<unsigned>(div_up(columns, 256))), dim3(256), 0, st, static_cast<const T *>(D.dy),
                                       D.dy_stride, static_cast<const T *>(D.y), static_cast<const unsigned char *>(D.mask), mask_pitch(D.c_out), dz,
                                       D.dbias ? partial : nullptr, D.offsets, n, D.experts, D.c_out, plan.dz_rows));
        return SPIRA_B200_OK;
      };
      const int kind = !D.relu ? 0 : D.mask ? 1 : 2;
      if (wide) rc = kind == 0 ? go(grouped_dz_kernel<T, 8, 0>, D.c_out / 8) : kind == 1 ? go(grouped_dz_kernel<T, 8, 1>, D.c_out / 8) : go(grouped_dz_kernel<T, 8, 2>, D.c_out / 8);
      else rc = kind == 0 ? go(grouped_dz_kernel<T, 1, 0>, D.c_out) : kind == 1 ? go(grouped_dz_kernel<T, 1, 1>, D.c_out) : go(grouped_dz_kernel<T, 1, 2>, D.c_out);
      if (rc != SPIRA_B200_OK) return rc;
      if (D.dbias)
        SB_CHECK_CUDA(launch_dependent(grouped_column_sum_kernel<T>, dim3(static_cast<unsigned>(div_up(D.c_out, 32)), D.experts), dim3(1024), 0, st,
                                       static_cast<const float *>(partial), D.offsets, n, D.experts, plan.dz_rows, D.c_out, static_cast<T *>(D.dbias)));
    }
    if (D.dx) {
      if (tc_dx(Z)) {
        rc = grouped_tc_run(kDx, Z, 0, nullptr, status, wait_ns(), st);
      } else {
        GroupedParams P{Z.dy, Z.weight, nullptr, Z.offsets, Z.dx, nullptr, Z.dy_stride, 0, n, Z.experts, Z.c_in, Z.c_out, 0, 0};
        rc = launch_any<T, kDx>(P, st);
      }
      if (rc != SPIRA_B200_OK) return rc;
    }
    if (!D.dweight) return SPIRA_B200_OK;
    if (tc_dw(Z)) {
      rc = grouped_tc_run(kDw, Z, plan.dw_rows, partial, status, wait_ns(), st);
    } else {
      GroupedParams P{Z.x, Z.dy, nullptr, Z.offsets, Z.dweight, partial, Z.x_stride, Z.dy_stride, n, Z.experts, Z.c_in, Z.c_out, 0, plan.dw_rows};
      rc = launch_any<T, kDw>(P, st);
    }
    if (rc != SPIRA_B200_OK || plan.dw_rows == 0) return rc;
    const unsigned blocks = static_cast<unsigned>(div_up(size, 256) < 1024 ? div_up(size, 256) : 1024);
    SB_CHECK_CUDA(launch_dependent(grouped_sum_kernel<T>, dim3(blocks, D.experts), dim3(256), 0, st, static_cast<const float *>(partial), D.offsets, n,
                                   D.experts, plan.dw_rows, size, static_cast<T *>(D.dweight)));
    return SPIRA_B200_OK;
  });
}
