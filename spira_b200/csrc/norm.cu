// Norms before and after a block, fused with the block's gate and the residual:
//
//   p = norm(block) * post_weight + post_bias          (or p = block)
//   stream = residual_scale * x + block_scale * gate * p
//   normed = norm(stream) * weight + bias
//   norm(v) = v / sqrt(mean(v^2) + eps)                (rms)
//           = (v - mean(v)) / sqrt(var(v) + eps)       (layer)
//
// Every row is read once and held in registers as fp32 from the first load to the last store: `normed` is the norm of the
// fp32 stream, not of its rounding.  The variance is the mean of squared differences (two sums over registers, no
// cancellation).  The backward pass reads x, block and the gate again and rebuilds the stream in fp32 from them and from
// the saved row statistics, so it needs neither output of the forward pass.  Parameter gradients are column sums: a thread
// owns its columns for all rows its CTA visits, CTAs write partial sums, a second launch adds those in a fixed order.
// Bound by memory: forward 2 row reads + 2 row writes, backward 4 + 2 (one more of each with a gate per element).
#include "common.cuh"
#include "elem.cuh"

namespace sb {

constexpr int kNormMaxChannels = 8192;
constexpr int kGateNone = 0, kGateChannel = 1, kGateRow = 2, kGateFull = 3;
constexpr int kNormBackwardCtas = 3;     // per SM at most: every CTA writes one set of partial sums
constexpr int kSums = 5;      // weight, bias, post_weight, post_bias, gate

struct NormParams {
  const void *x, *block, *gate, *dstream, *dnormed;
  const void *weight, *bias, *post_weight, *post_bias;
  void *stream, *normed, *dx, *dblock, *dgate;
  float *stats;               // [n][4]: mean and 1/deviation of the block, mean and 1/deviation of the stream
  float *partial;             // [CTAs][kSums][channels]
  int64_t n, x_stride, block_stride, gate_stride, dstream_stride, dnormed_stride;
  int channels, layer, pre, post, gate_kind, params_f32;
  float residual_scale, block_scale, eps, inv_channels;
};

// V parameters from element `c` on, as fp32 (parameters are stored in the rows' type or in fp32).
template <typename T, int V>
__device__ __forceinline__ void load_param(const void *p, int f32, int c, float (&f)[V]) {
  if (f32) {
    const float *s = static_cast<const float *>(p) + c;
    if constexpr (V % 4 == 0) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 q = *reinterpret_cast<const float4 *>(s + i);
        f[i] = q.x; f[i + 1] = q.y; f[i + 2] = q.z; f[i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = s[i];
    }
  } else {
    load_f32<T, V>(static_cast<const T *>(p) + c, f);
  }
}

// Sum over the L threads of a row: lanes of a warp (L <= 32) or all threads of the CTA.  Every thread gets the same value.
template <int L, int M>
__device__ __forceinline__ void row_sums(float (&v)[M], float *scratch) {
  constexpr int W = L < 32 ? L : 32;
#pragma unroll
  for (int d = 1; d < W; d *= 2)
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], d, W);
  if constexpr (L > 32) {
    constexpr int kWarps = L / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int m = 0; m < M; ++m) scratch[m * kWarps + warp] = v[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      v[m] = lane < kWarps ? scratch[m * kWarps + lane] : 0.f;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) v[m] += __shfl_xor_sync(0xffffffffu, v[m], d);
    }
    __syncthreads();
  }
}

// f = w * f + b with what there is of the two parameters
template <typename T, int V>
__device__ __forceinline__ void affine(const void *w, const void *b, int f32, int c, float (&f)[V]) {
  float q[V];
  if (w) {
    load_param<T, V>(w, f32, c, q);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] *= q[e];
  }
  if (b) {
    load_param<T, V>(b, f32, c, q);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] += q[e];
  }
}

// v becomes (v - mean) / deviation; st gets the mean and 1 / deviation.  Pieces outside the row are skipped.
template <int L, int ITEMS, int V, bool LAYER>
__device__ __forceinline__ void normalise(float (&v)[ITEMS][V], const bool (&in)[ITEMS], const NormParams &P, float *scratch, float &mean, float &r) {
  float s[1] = {0.f};
  if (LAYER) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (in[i])
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += v[i][e];
    row_sums<L, 1>(s, scratch);
    mean = s[0] * P.inv_channels;
    s[0] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (in[i])
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (LAYER) v[i][e] -= mean;
        s[0] = fmaf(v[i][e], v[i][e], s[0]);
      }
  row_sums<L, 1>(s, scratch);
  r = rsqrtf(fmaf(s[0], P.inv_channels, P.eps));
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) v[i][e] *= r;
}

// Threads of a CTA: 256, or the row's if it takes more.
template <int L>
constexpr int kNormThreads = L > 256 ? L : 256;

// L threads per row, each with ITEMS pieces of V neighbouring channels, L pieces apart.  What limits these kernels is not
// memory alone but instructions (20 to 40 per element against 8 to 14 bytes): options are tested per row and never per
// element, conversions work on pairs.
template <typename T, int V, int L, int ITEMS, bool LAYER>
__global__ void __launch_bounds__(kNormThreads<L>, L > 32 || ITEMS > 1 ? 1 : 4) norm_forward_kernel(const __grid_constant__ NormParams P) {
  __shared__ float scratch[32];
  pdl_trigger();
  pdl_wait();
  const int g = threadIdx.x % L;
  constexpr int kRows = kNormThreads<L> / L;
  const int64_t rounds = (P.n + kRows - 1) / kRows;
  bool in[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) in[i] = (i * L + g) * V < P.channels;
  for (int64_t b = blockIdx.x; b < rounds; b += gridDim.x) {
    const int64_t row = b * kRows + threadIdx.x / L;
    const bool live = row < P.n;
    float x[ITEMS][V] = {}, p[ITEMS][V] = {};
    Vec<T, V> gates[ITEMS];
    float row_gate = P.block_scale;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (live && in[i]) {
        const int c = (i * L + g) * V;
        load_f32<T, V>(static_cast<const T *>(P.x) + row * P.x_stride + c, x[i]);
        if (P.block) load_f32<T, V>(static_cast<const T *>(P.block) + row * P.block_stride + c, p[i]);
        if (P.gate_kind == kGateFull) gates[i] = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(P.gate) + row * P.gate_stride + c);
      }
    if (P.gate_kind == kGateRow && live) row_gate *= to_f32(static_cast<const T *>(P.gate)[row * P.gate_stride]);
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (P.block) {
      if (P.post) {
        normalise<L, ITEMS, V, LAYER>(p, in, P, scratch, st.x, st.y);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
          if (in[i]) affine<T, V>(P.post_weight, P.post_bias, P.params_f32, (i * L + g) * V, p[i]);
      }
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (!in[i]) continue;
        const int c = (i * L + g) * V;
        if (P.gate_kind == kGateChannel) {
          affine<T, V>(P.gate, nullptr, P.params_f32, c, p[i]);
        } else if (P.gate_kind == kGateFull) {
          float f[V];
          vec_to_f32<T, V>(gates[i], f);
#pragma unroll
          for (int e = 0; e < V; ++e) p[i][e] *= f[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = fmaf(row_gate, p[i][e], P.residual_scale * x[i][e]);
        if (live) store_f32<T, V>(static_cast<T *>(P.stream) + row * P.channels + c, x[i]);
      }
    }
    if (P.pre) {
      normalise<L, ITEMS, V, LAYER>(x, in, P, scratch, st.z, st.w);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (!in[i]) continue;
        const int c = (i * L + g) * V;
        affine<T, V>(P.weight, P.bias, P.params_f32, c, x[i]);
        if (live) store_f32<T, V>(static_cast<T *>(P.normed) + row * P.channels + c, x[i]);
      }
    }
    if (P.stats && live && g == 0) reinterpret_cast<float4 *>(P.stats)[row] = st;
  }
}

template <typename T, int V, int L, int ITEMS, bool LAYER>
__global__ void __launch_bounds__(kNormThreads<L>, L > 32 || ITEMS > 1 ? 1 : 2) norm_backward_kernel(const __grid_constant__ NormParams P) {
  constexpr int kThreads = kNormThreads<L>;
  __shared__ float scratch[64];
  extern __shared__ float column_sums[];      // [kThreads / L][channels]
  pdl_trigger();
  pdl_wait();
  const int g = threadIdx.x % L;
  constexpr int kRows = kThreads / L;
  const int64_t rounds = (P.n + kRows - 1) / kRows;
  const float a = P.residual_scale, s = P.block_scale;
  const void *post_w = P.post ? P.post_weight : nullptr, *post_b = P.post ? P.post_bias : nullptr;
  bool in[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) in[i] = (i * L + g) * V < P.channels;
  float sum[kSums][ITEMS][V] = {};
  for (int64_t b = blockIdx.x; b < rounds; b += gridDim.x) {
    const int64_t row = b * kRows + threadIdx.x / L;
    const bool live = row < P.n;
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    // hat: x, then the stream's normalised value; bh: the block's normalised value (or the block); d: gradient of the stream
    float hat[ITEMS][V] = {}, bh[ITEMS][V] = {}, d[ITEMS][V] = {}, u[ITEMS][V] = {};
    Vec<T, V> gates[ITEMS];
    float row_gate = 1.f;
    if (live) {
      st = reinterpret_cast<const float4 *>(P.stats)[row];
      if (P.gate_kind == kGateRow) row_gate = to_f32(static_cast<const T *>(P.gate)[row * P.gate_stride]);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (live && in[i]) {
        const int c = (i * L + g) * V;
        if (P.pre) {
          load_f32<T, V>(static_cast<const T *>(P.x) + row * P.x_stride + c, hat[i]);
          load_f32<T, V>(static_cast<const T *>(P.dnormed) + row * P.dnormed_stride + c, u[i]);
        }
        if (P.block) load_f32<T, V>(static_cast<const T *>(P.block) + row * P.block_stride + c, bh[i]);
        if (P.dstream) load_f32<T, V>(static_cast<const T *>(P.dstream) + row * P.dstream_stride + c, d[i]);
        if (P.gate_kind == kGateFull) gates[i] = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(P.gate) + row * P.gate_stride + c);
      }
    float sums[2] = {0.f, 0.f};
    if (P.post) {
      const float shift = -st.x * st.y;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) bh[i][e] = LAYER ? fmaf(bh[i][e], st.y, shift) : bh[i][e] * st.y;
    }
    // the factor of the block's value in the stream without block_scale
    auto load_gate = [&](int i, int c, float (&f)[V]) {
      if (P.gate_kind == kGateChannel) load_param<T, V>(P.gate, P.params_f32, c, f);
      else if (P.gate_kind == kGateFull && live) vec_to_f32<T, V>(gates[i], f);
      else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = row_gate;
      }
    };
    if (P.pre) {
      const float shift = -st.z * st.w;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (!in[i]) continue;
        const int c = (i * L + g) * V;
        if (P.block) {
          float q[V], f[V];
#pragma unroll
          for (int e = 0; e < V; ++e) q[e] = bh[i][e];
          affine<T, V>(post_w, post_b, P.params_f32, c, q);
          if (P.gate_kind != kGateNone) {
            load_gate(i, c, f);
#pragma unroll
            for (int e = 0; e < V; ++e) q[e] *= f[e];
          }
#pragma unroll
          for (int e = 0; e < V; ++e) hat[i][e] = fmaf(s, q[e], a * hat[i][e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          hat[i][e] = LAYER ? fmaf(hat[i][e], st.w, shift) : hat[i][e] * st.w;
          sum[0][i][e] = fmaf(u[i][e], hat[i][e], sum[0][i][e]);
          sum[1][i][e] += u[i][e];
        }
        affine<T, V>(P.weight, nullptr, P.params_f32, c, u[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sums[0] = fmaf(u[i][e], hat[i][e], sums[0]);
          if (LAYER) sums[1] += u[i][e];
        }
      }
      row_sums<L, 2>(sums, scratch);
      const float m0 = -sums[0] * P.inv_channels * st.w, m1 = LAYER ? -sums[1] * P.inv_channels * st.w : 0.f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          d[i][e] = fmaf(u[i][e], st.w, d[i][e]);
          d[i][e] = fmaf(hat[i][e], m0, d[i][e]);
          if (LAYER) d[i][e] += m1;
        }
    }
    if (live && P.dx)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (in[i]) {
          float o[V];
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] = P.block ? a * d[i][e] : d[i][e];
          store_f32<T, V>(static_cast<T *>(P.dx) + row * P.channels + (i * L + g) * V, o);
        }
    if (P.block) {
      sums[0] = sums[1] = 0.f;
      float gate_sum[1] = {0.f};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (!in[i]) continue;
        const int c = (i * L + g) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) d[i][e] *= s;
        if (P.gate_kind != kGateNone) {
          float q[V], f[V];
          load_gate(i, c, f);
          if (P.dgate) {
#pragma unroll
            for (int e = 0; e < V; ++e) q[e] = bh[i][e];
            affine<T, V>(post_w, post_b, P.params_f32, c, q);
#pragma unroll
            for (int e = 0; e < V; ++e) q[e] *= d[i][e];
            if (P.gate_kind == kGateChannel) {
#pragma unroll
              for (int e = 0; e < V; ++e) sum[4][i][e] += q[e];
            } else if (P.gate_kind == kGateRow) {
#pragma unroll
              for (int e = 0; e < V; ++e) gate_sum[0] += q[e];
            } else if (live) {
              store_f32<T, V>(static_cast<T *>(P.dgate) + row * P.channels + c, q);
            }
          }
#pragma unroll
          for (int e = 0; e < V; ++e) d[i][e] *= f[e];
        }
        if (P.post) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sum[2][i][e] = fmaf(d[i][e], bh[i][e], sum[2][i][e]);
            sum[3][i][e] += d[i][e];
          }
          affine<T, V>(post_w, nullptr, P.params_f32, c, d[i]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sums[0] = fmaf(d[i][e], bh[i][e], sums[0]);
            if (LAYER) sums[1] += d[i][e];
          }
        }
      }
      if (P.gate_kind == kGateRow && P.dgate) {
        row_sums<L, 1>(gate_sum, scratch);
        if (live && g == 0) static_cast<T *>(P.dgate)[row] = from_f32<T>(gate_sum[0]);
      }
      if (P.dblock) {
        if (P.post) {
          row_sums<L, 2>(sums, scratch);
          const float m0 = -sums[0] * P.inv_channels, m1 = LAYER ? -sums[1] * P.inv_channels : 0.f;
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) d[i][e] = st.y * fmaf(bh[i][e], m0, LAYER ? d[i][e] + m1 : d[i][e]);
        }
        if (live)
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
            if (in[i]) store_f32<T, V>(static_cast<T *>(P.dblock) + row * P.channels + (i * L + g) * V, d[i]);
      }
    }
  }
  if (P.partial == nullptr) return;
  // the CTA's column sums, rows of the CTA added in order
  const bool wanted[kSums] = {P.pre != 0 && P.weight, P.pre != 0 && P.bias, P.post != 0 && P.post_weight, P.post != 0 && P.post_bias,
                              P.gate_kind == kGateChannel};
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    if (!wanted[k]) continue;
    float *dst = P.partial + (static_cast<int64_t>(blockIdx.x) * kSums + k) * P.channels;
    if constexpr (kRows == 1) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (in[i])
#pragma unroll
          for (int e = 0; e < V; ++e) dst[(i * L + g) * V + e] = sum[k][i][e];
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (in[i])
#pragma unroll
          for (int e = 0; e < V; ++e) column_sums[(threadIdx.x / L) * P.channels + (i * L + g) * V + e] = sum[k][i][e];
      __syncthreads();
      for (int c = threadIdx.x; c < P.channels; c += kThreads) {
        float t = 0.f;
#pragma unroll 4
        for (int r = 0; r < kRows; ++r) t += column_sums[r * P.channels + c];
        dst[c] = t;
      }
    }
  }
}

struct NormSumParams {
  const float *partial;
  void *out[kSums];
  int ctas, channels, params_f32;
};

// out[k][c] = sum over CTAs: 32 columns x 32 strides of CTAs per block, then a fixed tree.
template <typename T>
__global__ void __launch_bounds__(1024) norm_sums_kernel(const __grid_constant__ NormSumParams P) {
  __shared__ float part[32][33];
  pdl_trigger();
  pdl_wait();
  const int k = blockIdx.y;
  if (P.out[k] == nullptr) return;
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < P.channels)
#pragma unroll 8
    for (int b = r; b < P.ctas; b += 32) t += P.partial[(static_cast<int64_t>(b) * kSums + k) * P.channels + c];
  part[r][lane] = t;
  __syncthreads();
  t = part[lane][r];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) t += __shfl_xor_sync(0xffffffffu, t, d);
  const int co = blockIdx.x * 32 + r;
  if (lane == 0 && co < P.channels) {
    if (P.params_f32) static_cast<float *>(P.out[k])[co] = t;
    else static_cast<T *>(P.out[k])[co] = from_f32<T>(t);
  }
}

// CTAs of a kernel that fit on an SM (asked once per kernel).
template <typename K>
static int resident_ctas(K kernel, int threads) {
  int n = 0;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) == cudaSuccess && n > 0 ? n : 1;
}

template <typename T, int V, int L, int ITEMS, bool LAYER>
static int launch_norm_kind(const NormParams &P, bool backward, int *ctas, cudaStream_t st) {
  constexpr int kThreads = kNormThreads<L>;
  constexpr int kRows = kThreads / L;
  const int64_t rounds = div_up(P.n, kRows);
  if (!backward) {
    static const int resident = resident_ctas(norm_forward_kernel<T, V, L, ITEMS, LAYER>, kThreads);
    const int64_t cap = static_cast<int64_t>(sm_count()) * resident;
    SB_CHECK_CUDA(launch_dependent(norm_forward_kernel<T, V, L, ITEMS, LAYER>, dim3(static_cast<unsigned>(rounds < cap ? rounds : cap)), dim3(kThreads), 0,
                                   st, P));
    return SPIRA_B200_OK;
  }
  static const int resident = resident_ctas(norm_backward_kernel<T, V, L, ITEMS, LAYER>, kThreads);
  const int64_t cap = static_cast<int64_t>(sm_count()) * (resident < kNormBackwardCtas ? resident : kNormBackwardCtas);
  const int grid = static_cast<int>(rounds < cap ? rounds : cap);
  *ctas = grid;
  const size_t smem = kRows > 1 ? static_cast<size_t>(kRows) * P.channels * 4 : 0;
  SB_CHECK_CUDA(launch_dependent(norm_backward_kernel<T, V, L, ITEMS, LAYER>, dim3(grid), dim3(kThreads), smem, st, P));
  return SPIRA_B200_OK;
}

template <typename T, int V, int L, int ITEMS>
static int launch_norm(const NormParams &P, bool backward, int *ctas, cudaStream_t st) {
  return P.layer ? launch_norm_kind<T, V, L, ITEMS, true>(P, backward, ctas, st) : launch_norm_kind<T, V, L, ITEMS, false>(P, backward, ctas, st);
}

// Threads per row and pieces per thread: the fewest lanes that hold the row, so that a row sum takes few shuffles; rows too
// long for a warp's registers take a whole CTA.
template <typename T, int V>
static int launch_norm_shape(const NormParams &P, bool backward, int *ctas, cudaStream_t st) {
  const int pieces = P.channels / V;
  if constexpr (V > 1) {
    if (pieces <= 4) return launch_norm<T, V, 4, 1>(P, backward, ctas, st);
    if (pieces <= 8) return launch_norm<T, V, 8, 1>(P, backward, ctas, st);
    if (pieces <= 16) return launch_norm<T, V, 16, 1>(P, backward, ctas, st);
  }
  if (pieces <= 32) return launch_norm<T, V, 32, 1>(P, backward, ctas, st);
  if (pieces <= 64) return launch_norm<T, V, 32, 2>(P, backward, ctas, st);
  if (pieces <= 256) return launch_norm<T, V, 256, 1>(P, backward, ctas, st);
  if (pieces <= 512) return launch_norm<T, V, 256, 2>(P, backward, ctas, st);
  if constexpr (V == 8) {
    return launch_norm<T, V, 512, 2>(P, backward, ctas, st);       // (8192 channels are 1024 pieces)
  } else {
    if (pieces <= 1024) return launch_norm<T, V, 512, 2>(P, backward, ctas, st);
    if constexpr (V == 1) {
      if (pieces > 4096) return launch_norm<T, V, 1024, 8>(P, backward, ctas, st);
      if (pieces > 2048) return launch_norm<T, V, 1024, 4>(P, backward, ctas, st);
    }
    return launch_norm<T, V, 1024, 2>(P, backward, ctas, st);
  }
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool norm_wide(const spira_b200_norm_desc &D, int size) {
  auto rows = [&](const void *p, int64_t stride) { return p == nullptr || (aligned16(p) && stride * size % 16 == 0); };
  return D.channels * size % 16 == 0 && rows(D.x, D.x_stride) && rows(D.block, D.block_stride) && rows(D.dstream, D.dstream_stride) &&
         rows(D.dnormed, D.dnormed_stride) && (D.gate_kind == kGateRow || rows(D.gate, D.gate_kind == kGateFull ? D.gate_stride : 0)) &&
         rows(D.stream, 0) && rows(D.normed, 0) && rows(D.dx, 0) && rows(D.dblock, 0) && (D.gate_kind != kGateFull || rows(D.dgate, 0)) &&
         aligned16(D.weight) && aligned16(D.bias) && aligned16(D.post_weight) && aligned16(D.post_bias);
}

static int norm_check(const char *what, const spira_b200_norm_desc *D) {
  SB_CHECK_ARG(D, "%s: null descriptor", what);
  SB_CHECK_ARG(D->dtype >= SPIRA_B200_F16 && D->dtype <= SPIRA_B200_F32, "%s: unknown element type %d", what, D->dtype);
  SB_CHECK_ARG(D->n >= 0 && D->n < (int64_t(1) << 31), "%s: n=%lld out of range", what, (long long)D->n);
  SB_CHECK_ARG(D->channels >= 1 && D->channels <= kNormMaxChannels, "%s: channels=%d must be 1 to %d", what, D->channels, kNormMaxChannels);
  SB_CHECK_ARG(D->gate_kind >= kGateNone && D->gate_kind <= kGateFull, "%s: unknown gate %d", what, D->gate_kind);
  SB_CHECK_ARG(D->eps > 0.f, "%s: eps must be positive", what);
  SB_CHECK_ARG(D->x_stride >= 0 && D->block_stride >= 0 && D->gate_stride >= 0 && D->dstream_stride >= 0 && D->dnormed_stride >= 0,
               "%s: negative row stride", what);
  if (D->n == 0) return SPIRA_B200_OK;      // (tensors without rows have no address)
  SB_CHECK_ARG(D->pre || D->block, "%s: neither a block nor a norm", what);
  SB_CHECK_ARG(D->block || (!D->post && D->gate_kind == kGateNone), "%s: a gate or a norm after the block needs a block", what);
  SB_CHECK_ARG((D->gate_kind == kGateNone) == (D->gate == nullptr), "%s: gate and its kind do not match", what);
  return SPIRA_B200_OK;
}

static NormParams norm_params(const spira_b200_norm_desc &D) {
  NormParams P{};
  P.x = D.x; P.block = D.block; P.gate = D.gate; P.dstream = D.dstream; P.dnormed = D.dnormed;
  P.weight = D.weight; P.bias = D.bias; P.post_weight = D.post_weight; P.post_bias = D.post_bias;
  P.stream = D.stream; P.normed = D.normed; P.dx = D.dx; P.dblock = D.dblock; P.dgate = D.dgate;
  P.stats = D.stats;
  P.n = D.n; P.x_stride = D.x_stride; P.block_stride = D.block_stride; P.gate_stride = D.gate_stride;
  P.dstream_stride = D.dstream_stride; P.dnormed_stride = D.dnormed_stride;
  P.channels = D.channels; P.layer = D.layer; P.pre = D.pre; P.post = D.post; P.gate_kind = D.gate_kind; P.params_f32 = D.params_f32;
  P.residual_scale = D.residual_scale; P.block_scale = D.block_scale; P.eps = D.eps; P.inv_channels = 1.f / static_cast<float>(D.channels);
  return P;
}

static int norm_run(const spira_b200_norm_desc &D, const NormParams &P, bool backward, int *ctas, cudaStream_t st) {
  const bool wide = norm_wide(D, elem_size(D.dtype));
  return SB_DISPATCH_ELEM(D.dtype, T, {
    if (wide) return launch_norm_shape<T, 16 / static_cast<int>(sizeof(T))>(P, backward, ctas, st);
    return launch_norm_shape<T, 1>(P, backward, ctas, st);
  });
}

}  // namespace sb

using namespace sb;

extern "C" int spira_b200_residual_norm(const spira_b200_norm_desc *desc, void *stream) {
  int rc = norm_check("residual_norm", desc);
  if (rc != SPIRA_B200_OK || desc->n == 0) return rc;
  SB_CHECK_ARG(desc->x && (!desc->pre || desc->normed) && (!desc->block || desc->stream), "residual_norm: null pointer");
  return norm_run(*desc, norm_params(*desc), false, nullptr, as_stream(stream));
}

extern "C" int spira_b200_residual_norm_backward_workspace(const spira_b200_norm_desc *desc, size_t *bytes) {
  int rc = norm_check("residual_norm_backward", desc);
  if (rc != SPIRA_B200_OK) return rc;
  SB_CHECK_ARG(bytes, "residual_norm_backward: null pointer");
  *bytes = static_cast<size_t>(sm_count()) * kNormBackwardCtas * kSums * desc->channels * 4;
  return SPIRA_B200_OK;
}

extern "C" int spira_b200_residual_norm_backward(const spira_b200_norm_desc *desc, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = norm_check("residual_norm_backward", desc);
  if (rc != SPIRA_B200_OK) return rc;
  const spira_b200_norm_desc &D = *desc;
  const bool sums = D.dweight || D.dbias || D.dpost_weight || D.dpost_bias || (D.gate_kind == kGateChannel && D.dgate);
  SB_CHECK_ARG(D.n == 0 || (D.stats && (!D.pre || (D.x && D.dnormed)) && (D.dstream || D.pre)), "residual_norm_backward: null pointer");
  SB_CHECK_ARG((!D.dweight || D.weight) && (!D.dbias || D.bias) && (!D.dpost_weight || D.post_weight) && (!D.dpost_bias || D.post_bias),
               "residual_norm_backward: the gradient of a parameter that is not there");
  NormParams P = norm_params(D);
  size_t need = 0;
  rc = spira_b200_residual_norm_backward_workspace(desc, &need);
  if (rc != SPIRA_B200_OK) return rc;
  if (sums) {
    if (workspace == nullptr || workspace_bytes < need)
      return fail(SPIRA_B200_ERR_WORKSPACE, "residual_norm_backward: workspace of %zu bytes is smaller than %zu", workspace_bytes, need);
    P.partial = static_cast<float *>(workspace);
  }
  cudaStream_t st = as_stream(stream);
  int ctas = 0;
  if (D.n > 0) {
    rc = norm_run(D, P, true, &ctas, st);
    if (rc != SPIRA_B200_OK) return rc;
  }
  if (!sums) return SPIRA_B200_OK;
  NormSumParams S{};
  S.partial = P.partial;
  S.out[0] = D.dweight; S.out[1] = D.dbias; S.out[2] = D.dpost_weight; S.out[3] = D.dpost_bias;
  S.out[4] = D.gate_kind == kGateChannel ? D.dgate : nullptr;
  S.ctas = ctas; S.channels = D.channels; S.params_f32 = D.params_f32;
  return SB_DISPATCH_ELEM(D.dtype, T, {
    SB_CHECK_CUDA(launch_dependent(norm_sums_kernel<T>, dim3(static_cast<unsigned>(div_up(D.channels, 32)), kSums), dim3(1024), 0, st, S));
    return SPIRA_B200_OK;
  });
}
