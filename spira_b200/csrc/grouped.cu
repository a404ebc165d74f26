// Ragged products of grouped rows with one weight matrix per group (the experts of a mixture):
//
//   y[r]  = relu?(x[r] W[e] + b[e])      rows r of group e
//   dz    = dy (y > 0)                    db[e] = sum over the group's rows of dz
//   dx[r] = dz[r] W[e]^T                  dW[e] = x_e^T dz_e
//
// Rows outside every group are zero in y and dx.  Group boundaries are read on the device; the host only knows upper
// bounds of the tile counts.  Sums over a group's rows are split into pieces that are added in a fixed order.
//
// Products run on the tensor-core kernel (grouped_tc.cu), which wants rows on 16-byte boundaries.  Channel counts, strides or
// addresses that break them are met in two ways: large products copy what is off into rows of a pitch in whole units of 8
// (and their result back), small ones run on `grouped_any_kernel`, which takes everything: 64 x 64 tiles, element-wise loads
// into shared memory, warp-level MMAs with fp32 accumulation.
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
  unsigned char *mask;            // forward: a bit per element that the ReLU let through
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
      k_end = piece_end(k_begin, t.end, P.piece);
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
    for (int j = 0; j < 4; ++j) {
      uint32_t bits[2] = {0, 0};                      // of rows g and g + 8: two columns of this lane's, of a byte
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = m0 + wm + 16 * i + g + 8 * (q >> 1), n = n0 + wn + 8 * j + 2 * t4 + (q & 1);
        if (m >= m_end || n >= n_end) continue;
        float v = acc[i][j][q];
        if (MODE == kForward) {
          if (P.bias) v += to_f32(static_cast<const T *>(P.bias)[static_cast<int64_t>(expert) * P.c_out + n]);
          if (v > 0.f) bits[q >> 1] |= 1u << (2 * t4 + (q & 1));
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
      if (MODE == kForward && P.mask) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          bits[h] |= __shfl_xor_sync(0xffffffffu, bits[h], 1);
          bits[h] |= __shfl_xor_sync(0xffffffffu, bits[h], 2);
          const int m = m0 + wm + 16 * i + g + 8 * h, n = n0 + wn + 8 * j;
          if (t4 == 0 && m < m_end && n < n_end) P.mask[static_cast<int64_t>(m) * mask_pitch(P.c_out) + n / 8] = static_cast<unsigned char>(bits[h]);
        }
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
    const int mine = i <= e ? pieces_of(hi - lo, piece) : 0;
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

// out[e][row][c] = sum over the pieces of group e, in order, of partial[piece][row][c]; rows of the partial sums are `pitch` long
template <typename T>
__global__ void __launch_bounds__(256) grouped_sum_kernel(const float *partial, const int32_t *offsets, int n, int experts, int piece, int64_t rows, int columns,
                                                          int pitch, T *out) {
  pdl_trigger();
  pdl_wait();
  const int e = blockIdx.y;
  int64_t first;
  int count;
  group_pieces(offsets, n, e, piece, first, count);
  const int64_t size = rows * pitch;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < size; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / pitch;
    const int c = static_cast<int>(i - row * pitch);
    if (c >= columns) continue;
    float t = 0.f;
#pragma unroll 4
    for (int p = 0; p < count; ++p) t += partial[(first + p) * size + i];
    out[(e * rows + row) * columns + c] = from_f32<T>(t);
  }
}

// Rows of one pitch into rows of another (16-bit elements): neighbouring threads take neighbouring elements, four per thread
// in flight.  Rows in groups of less than 2^31 elements (blockIdx.y), divided by multiplication.
struct RepitchParams {
  const unsigned short *src;
  unsigned short *dst;
  int64_t src_pitch, dst_pitch, rows, rows_per_group;
  int columns, div_shift;
  uint64_t div_mul;
};

__global__ void __launch_bounds__(256) grouped_repitch_kernel(const __grid_constant__ RepitchParams P) {
  pdl_trigger();
  pdl_wait();
  const int64_t row0 = blockIdx.y * P.rows_per_group;
  const int64_t here = P.rows - row0 < P.rows_per_group ? P.rows - row0 : P.rows_per_group;
  const uint32_t count = static_cast<uint32_t>(here * P.columns), first = blockIdx.x * 1024u + threadIdx.x;
  unsigned short v[4];
  int64_t to[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t i = first + 256u * q;
    if (i < count) {
      const uint32_t r = static_cast<uint32_t>((i * P.div_mul) >> P.div_shift), c = i - r * static_cast<uint32_t>(P.columns);
      v[q] = P.src[(row0 + r) * P.src_pitch + c];
      to[q] = (row0 + r) * P.dst_pitch + c;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (first + 256u * q < count) P.dst[to[q]] = v[q];
}

// dz = dy where the ReLU let the value through (dz != NULL), and column sums over pieces of a group's rows.  What the ReLU
// let through: MASK 1 a bit per element that the forward pass wrote, 2 y > 0, 0 everything (no ReLU).  A copy with four
// rows of a thread in flight; four CTAs per SM.
template <typename T, int V, int MASK>
__global__ void __launch_bounds__(256, 4) grouped_dz_kernel(const T *dy, int64_t dy_stride, const T *y, const unsigned char *mask, int mask_pitch, T *dz,
                                                            int64_t dz_pitch, float *partial, const int32_t *offsets, int n, int experts, int c_out, int piece) {
  __shared__ float sums[256 * V];
  pdl_trigger();
  pdl_wait();
  const GroupTile t = find_group_tile(offsets, experts, n, piece, blockIdx.x);
  if (t.expert < 0) return;
  const int r0 = t.begin + t.index * piece, r1 = piece_end(r0, t.end, piece);
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
        if (dz) *reinterpret_cast<Vec<T, V> *>(dz + row * dz_pitch + c) = d[q];
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

// Column sums of many short pieces: 32 columns x 8 strides of pieces per block, then a fixed order.  Latency of the
// loads: 64 x 16 blocks over 600 pieces 7.3 us; with 32 strides (1024 threads, two blocks per SM at a time) 12.1 us.
template <typename T>
__global__ void __launch_bounds__(256) grouped_column_sum_kernel(const float *partial, const int32_t *offsets, int n, int experts, int piece, int size, T *out) {
  __shared__ float part[8][32];
  pdl_trigger();
  pdl_wait();
  const int e = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  int64_t first;
  int count;
  group_pieces(offsets, n, e, piece, first, count);
  float t = 0.f;
  if (c < size)
#pragma unroll 8
    for (int p = w; p < count; p += 8) t += partial[(first + p) * size + c];
  part[w][lane] = t;
  __syncthreads();
  if (w == 0 && c < size) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += part[i][lane];
    out[static_cast<int64_t>(e) * size + c] = from_f32<T>(t);
  }
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

// Whether a product that needs copies for the tensor cores is worth them: 2^28 multiply-adds take the general kernel about
// 11 us, the copies and their launches 5 to 10; measured 20 000 rows 501 -> 703: 217 us without, 67 us with copies.
// With few rows per group the copy of the weights would outweigh the product.
static bool worth_copies(const spira_b200_grouped_desc &D) {
  return D.n * D.c_in >= (int64_t(1) << 28) / D.c_out && D.n >= 16 * static_cast<int64_t>(D.experts);
}

static unsigned long long wait_ns() { return static_cast<unsigned long long>(spira_b200_get_option("wait_limit_us")) * 1000ull; }

static int64_t any_tiles(int c_in, int c_out) { return div_up(c_in, kATile) * div_up(c_out, kATile); }

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
  SB_CHECK_CUDA(launch_operator(grouped_any_kernel<T, MODE>, dim3(static_cast<unsigned>(units < 1 ? 1 : units), static_cast<unsigned>(columns)),
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

// A scratch plan hands out 256-byte aligned places.
struct Scratch {
  size_t bytes = 0;
  size_t take(int64_t want) {
    const size_t at = bytes;
    bytes += (static_cast<size_t>(want) + 255) / 256 * 256;
    return at;
  }
};
constexpr size_t kNoCopy = ~size_t(0);

struct ForwardPlan {
  bool tc;
  size_t x, w, y;        // where their copies lie, or kNoCopy
  size_t bytes;
};

static ForwardPlan forward_plan(const spira_b200_grouped_desc &D) {
  ForwardPlan p{false, kNoCopy, kNoCopy, kNoCopy, 0};
  const bool x_ok = grouped_tc_rows_ok(D.x, D.x_stride, D.c_in, D.n), even = D.c_out % 8 == 0;
  const bool w_ok = even && aligned16(D.weight), y_ok = even && aligned16(D.y);
  p.tc = grouped_tc_available() && ((x_ok && w_ok && y_ok) || worth_copies(D));
  if (!p.tc) return p;
  Scratch s;
  if (!x_ok) p.x = s.take(D.n * pitch8(D.c_in) * 2);
  if (!w_ok) p.w = s.take(static_cast<int64_t>(D.experts) * D.c_in * pitch8(D.c_out) * 2);
  if (!y_ok) p.y = s.take(D.n * pitch8(D.c_out) * 2);
  p.bytes = s.bytes;
  return p;
}

static int repitch(const void *src, int64_t src_pitch, void *dst, int64_t dst_pitch, int64_t rows, int columns, cudaStream_t st) {
  RepitchParams P{static_cast<const unsigned short *>(src), static_cast<unsigned short *>(dst), src_pitch, dst_pitch, rows, 0, columns, 0, 0};
  P.rows_per_group = ((int64_t(1) << 31) - 2048) / columns;
  if (P.rows_per_group > rows) P.rows_per_group = rows;
  int bits = 0;
  while ((int64_t(1) << bits) < columns) ++bits;
  P.div_shift = 31 + bits;
  P.div_mul = ((uint64_t(1) << P.div_shift) + columns - 1) / columns;
  const dim3 grid(static_cast<unsigned>(div_up(P.rows_per_group * columns, 1024)), static_cast<unsigned>(div_up(rows, P.rows_per_group)));
  SB_CHECK_CUDA(launch_operator(grouped_repitch_kernel, grid, dim3(256), 0, st, P));
  return SPIRA_B200_OK;
}

static int check_workspace(const char *what, const void *workspace, size_t have, size_t need) {
  if (need && (!workspace || have < need)) return fail(SPIRA_B200_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than %zu", what, have, need);
  SB_CHECK_ARG(need == 0 || aligned16(workspace), "%s: the workspace must be 16-byte aligned", what);
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_grouped_linear_workspace(const spira_b200_grouped_desc *desc, size_t *workspace_bytes, size_t *mask_bytes) {
  int rc = grouped_check("grouped_linear", desc);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(workspace_bytes && mask_bytes, "grouped_linear: null pointer");
  *workspace_bytes = *mask_bytes = 0;
  if (desc->n == 0) return SPIRA_B200_OK;
  const ForwardPlan plan = forward_plan(*desc);
  *workspace_bytes = plan.bytes;
  *mask_bytes = desc->relu ? static_cast<size_t>(desc->n) * mask_pitch(desc->c_out) : 0;
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_grouped_linear(const spira_b200_grouped_desc *desc, void *workspace, size_t workspace_bytes, int32_t *status, void *stream) {
  int rc = grouped_check("grouped_linear", desc);
  if (rc != SPIRA_B200_OK || desc->n == 0) return rc;
  const spira_b200_grouped_desc &D = *desc;
  SB_CHECK_ARG(D.x && D.weight && D.y, "grouped_linear: null pointer");
  const ForwardPlan plan = forward_plan(D);
  SB_CHECK_ARG(!D.mask || D.relu, "grouped_linear: no mask is written for this call (spira_b200_grouped_linear_workspace says 0)");
  cudaStream_t st = as_stream(stream);
  if (!plan.tc) {
    GroupedParams P{D.x, D.weight, D.bias, D.offsets, D.y, nullptr, D.x_stride, 0, static_cast<int>(D.n), D.experts, D.c_in, D.c_out, D.relu, 0,
                    static_cast<unsigned char *>(D.mask)};
    return SB_DISPATCH_HALF(D.dtype, T, return (launch_any<T, kForward>(P, st)););
  }
  rc = check_workspace("grouped_linear", workspace, workspace_bytes, plan.bytes);
  if (rc != SPIRA_B200_OK) return rc;
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  spira_b200_grouped_desc Z = D;
  int w_pitch = D.c_out, y_pitch = D.c_out;
  if (plan.x != kNoCopy) {
    Z.x = ws + plan.x;
    Z.x_stride = pitch8(D.c_in);
    rc = repitch(D.x, D.x_stride, ws + plan.x, Z.x_stride, D.n, D.c_in, st);
    if (rc != SPIRA_B200_OK) return rc;
  }
  if (plan.w != kNoCopy) {
    Z.weight = ws + plan.w;
    w_pitch = pitch8(D.c_out);
    rc = repitch(D.weight, D.c_out, ws + plan.w, w_pitch, static_cast<int64_t>(D.experts) * D.c_in, D.c_out, st);
    if (rc != SPIRA_B200_OK) return rc;
  }
  if (plan.y != kNoCopy) {
    Z.y = ws + plan.y;
    y_pitch = pitch8(D.c_out);
  }
  rc = grouped_tc_run(kForward, Z, w_pitch, y_pitch, 0, nullptr, status, wait_ns(), st);
  if (rc != SPIRA_B200_OK || plan.y == kNoCopy) return rc;
  return repitch(Z.y, y_pitch, D.y, D.c_out, D.n, D.c_out, st);
}

// The backward pass: dz (where a ReLU followed, or where dy itself is not fit for the tensor cores) and the column sums in
// one copy of dy, then dx and dW from it.  Copies as in the forward pass; the partial sums of dbias and of dweight follow
// one another in one place.
struct BackwardPlan {
  bool tc;
  size_t dz, x, w, dx, dw, partial;
  int64_t dz_pitch;
  int dz_rows, dw_rows;
  size_t bytes;
};

static BackwardPlan backward_plan(const spira_b200_grouped_desc &D) {
  BackwardPlan p{};
  const bool x_ok = !D.dweight || grouped_tc_rows_ok(D.x, D.x_stride, D.c_in, D.n), dy_ok = D.relu || grouped_tc_rows_ok(D.dy, D.dy_stride, D.c_out, D.n);
  const bool w_ok = !D.dx || (D.c_out % 8 == 0 && aligned16(D.weight)), dx_ok = !D.dx || (D.c_in % 8 == 0 && aligned16(D.dx));
  const bool dw_ok = !D.dweight || (D.c_out % 8 == 0 && aligned16(D.dweight));
  p.tc = grouped_tc_available() && ((x_ok && dy_ok && w_ok && dx_ok && dw_ok) || worth_copies(D));
  p.dz = p.x = p.w = p.dx = p.dw = kNoCopy;
  p.dz_rows = dz_piece(D.n);
  p.dz_pitch = pitch8(D.c_out);
  Scratch s;
  if ((D.dx || D.dweight) && (D.relu || (p.tc && !dy_ok))) p.dz = s.take(D.n * p.dz_pitch * 2);
  if (D.dweight)
    p.dw_rows = p.tc ? dw_piece(D.n, D.experts, grouped_tc_dw_tiles(D.c_in, D.c_out), 1) : dw_piece(D.n, D.experts, any_tiles(D.c_in, D.c_out), 2);
  if (p.tc) {
    if (!x_ok) p.x = s.take(D.n * pitch8(D.c_in) * 2);
    if (!w_ok) p.w = s.take(static_cast<int64_t>(D.experts) * D.c_in * pitch8(D.c_out) * 2);
    if (!dx_ok) p.dx = s.take(D.n * pitch8(D.c_in) * 2);
    if (!dw_ok && p.dw_rows == 0) p.dw = s.take(static_cast<int64_t>(D.experts) * D.c_in * pitch8(D.c_out) * 2);
  }
  const int64_t db = D.dbias ? group_tiles_bound(D.n, D.experts, p.dz_rows) * D.c_out * 4 : 0;
  const int64_t dw = p.dw_rows ? group_tiles_bound(D.n, D.experts, p.dw_rows) * D.c_in * (p.tc ? pitch8(D.c_out) : D.c_out) * 4 : 0;
  p.partial = s.take(db > dw ? db : dw);
  p.bytes = s.bytes;
  return p;
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
  *bytes = desc->n ? backward_plan(*desc).bytes : 0;
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_grouped_linear_paths(const spira_b200_grouped_desc *desc, int32_t *paths) {
  int rc = grouped_check("grouped_linear_paths", desc);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(paths && desc->n > 0, "grouped_linear_paths: null pointer, or no rows");
  const spira_b200_grouped_desc &D = *desc;
  auto path = [&](int mode, bool tc) { return !tc ? 0 : grouped_tc_pair(mode, D) ? 2 : 1; };
  const BackwardPlan plan = backward_plan(D);
  paths[0] = path(kForward, forward_plan(D).tc);
  paths[1] = D.dx ? path(kDx, plan.tc) : -1;
  paths[2] = D.dweight ? path(kDw, plan.tc) : -1;
  paths[3] = D.dweight ? plan.dw_rows : -1;
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_grouped_linear_backward(const spira_b200_grouped_desc *desc, void *workspace, size_t workspace_bytes, int32_t *status,
                                                  void *stream) {
  int rc = backward_check(desc);
  if (rc != SPIRA_B200_OK) return rc;
  const spira_b200_grouped_desc &D = *desc;
  cudaStream_t st = as_stream(stream);
  if (D.n == 0) {
    if (D.dweight) SB_CHECK_CUDA(cudaMemsetAsync(D.dweight, 0, static_cast<size_t>(D.experts) * D.c_in * D.c_out * 2, st));
    if (D.dbias) SB_CHECK_CUDA(cudaMemsetAsync(D.dbias, 0, static_cast<size_t>(D.experts) * D.c_out * 2, st));
    return SPIRA_B200_OK;
  }
  const BackwardPlan plan = backward_plan(D);
  rc = check_workspace("grouped_linear_backward", workspace, workspace_bytes, plan.bytes);
  if (rc != SPIRA_B200_OK) return rc;
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  float *partial = reinterpret_cast<float *>(ws + plan.partial);
  const int n = static_cast<int>(D.n);
  spira_b200_grouped_desc Z = D;
  return SB_DISPATCH_HALF(D.dtype, T, {
    if (plan.dz != kNoCopy || D.dbias) {
      T *dz = plan.dz != kNoCopy ? reinterpret_cast<T *>(ws + plan.dz) : nullptr;
      const unsigned units = static_cast<unsigned>(group_tiles_bound(n, D.experts, plan.dz_rows));
      const bool wide = D.c_out % 8 == 0 && aligned16(D.dy) && (D.dy_stride % 8 == 0 || n == 1) && (D.mask || aligned16(D.y));
      auto go = [&](auto kernel, int columns) -> int {
        SB_CHECK_CUDA(launch_operator(kernel, dim3(units, static_cast<unsigned>(div_up(columns, 256))), dim3(256), 0, st, static_cast<const T *>(D.dy),
                                       D.dy_stride, static_cast<const T *>(D.y), static_cast<const unsigned char *>(D.mask), mask_pitch(D.c_out), dz,
                                       plan.dz_pitch, D.dbias ? partial : nullptr, D.offsets, n, D.experts, D.c_out, plan.dz_rows));
        return SPIRA_B200_OK;
      };
      const int kind = !D.relu ? 0 : D.mask ? 1 : 2;
      if (wide) rc = kind == 0 ? go(grouped_dz_kernel<T, 8, 0>, D.c_out / 8) : kind == 1 ? go(grouped_dz_kernel<T, 8, 1>, D.c_out / 8) : go(grouped_dz_kernel<T, 8, 2>, D.c_out / 8);
      else rc = kind == 0 ? go(grouped_dz_kernel<T, 1, 0>, D.c_out) : kind == 1 ? go(grouped_dz_kernel<T, 1, 1>, D.c_out) : go(grouped_dz_kernel<T, 1, 2>, D.c_out);
      if (rc != SPIRA_B200_OK) return rc;
      if (D.dbias)
        SB_CHECK_CUDA(launch_operator(grouped_column_sum_kernel<T>, dim3(static_cast<unsigned>(div_up(D.c_out, 32)), D.experts), dim3(256), 0, st,
                                       static_cast<const float *>(partial), D.offsets, n, D.experts, plan.dz_rows, D.c_out, static_cast<T *>(D.dbias)));
      if (dz) {
        Z.dy = dz;
        Z.dy_stride = plan.dz_pitch;
      }
    }
    int w_pitch = D.c_out;
    const int dx_pitch = plan.dx != kNoCopy ? pitch8(D.c_in) : D.c_in, dw_pitch = plan.tc ? pitch8(D.c_out) : D.c_out;
    if (plan.x != kNoCopy) {
      Z.x = ws + plan.x;
      Z.x_stride = pitch8(D.c_in);
      rc = repitch(D.x, D.x_stride, ws + plan.x, Z.x_stride, D.n, D.c_in, st);
      if (rc != SPIRA_B200_OK) return rc;
    }
    if (plan.w != kNoCopy) {
      Z.weight = ws + plan.w;
      w_pitch = pitch8(D.c_out);
      rc = repitch(D.weight, D.c_out, ws + plan.w, w_pitch, static_cast<int64_t>(D.experts) * D.c_in, D.c_out, st);
      if (rc != SPIRA_B200_OK) return rc;
    }
    if (plan.dx != kNoCopy) Z.dx = ws + plan.dx;
    if (plan.dw != kNoCopy) Z.dweight = ws + plan.dw;
    if (D.dx) {
      if (plan.tc) {
        rc = grouped_tc_run(kDx, Z, w_pitch, dx_pitch, 0, nullptr, status, wait_ns(), st);
        if (rc == SPIRA_B200_OK && plan.dx != kNoCopy) rc = repitch(Z.dx, dx_pitch, D.dx, D.c_in, D.n, D.c_in, st);
      } else {
        GroupedParams P{Z.dy, Z.weight, nullptr, Z.offsets, Z.dx, nullptr, Z.dy_stride, 0, n, Z.experts, Z.c_in, Z.c_out, 0, 0, nullptr};
        rc = launch_any<T, kDx>(P, st);
      }
      if (rc != SPIRA_B200_OK) return rc;
    }
    if (!D.dweight) return SPIRA_B200_OK;
    if (plan.tc) {
      rc = grouped_tc_run(kDw, Z, w_pitch, dw_pitch, plan.dw_rows, partial, status, wait_ns(), st);
      if (rc == SPIRA_B200_OK && plan.dw != kNoCopy) rc = repitch(Z.dweight, dw_pitch, D.dweight, D.c_out, static_cast<int64_t>(D.experts) * D.c_in, D.c_out, st);
    } else {
      GroupedParams P{Z.x, Z.dy, nullptr, Z.offsets, Z.dweight, partial, Z.x_stride, Z.dy_stride, n, Z.experts, Z.c_in, Z.c_out, 0, plan.dw_rows, nullptr};
      rc = launch_any<T, kDw>(P, st);
    }
    if (rc != SPIRA_B200_OK || plan.dw_rows == 0) return rc;
    const int64_t want = div_up(static_cast<int64_t>(D.c_in) * dw_pitch, 256);
    SB_CHECK_CUDA(launch_operator(grouped_sum_kernel<T>, dim3(static_cast<unsigned>(want < 1024 ? want : 1024), D.experts), dim3(256), 0, st,
                                   static_cast<const float *>(partial), D.offsets, n, D.experts, plan.dw_rows, static_cast<int64_t>(D.c_in), D.c_out, dw_pitch,
                                   static_cast<T *>(D.dweight)));
    return SPIRA_B200_OK;
  });
}
