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
// Bound by memory and by the latency of a row's chain at the warps that registers leave room for: forward 2 row reads + 2 row writes, backward 4 + 2 (one more of each with a
// gate per element).  127 363 x 256 bf16, layer norms on both sides, a gate per element, fp32 parameters: forward 60 us =
// 5.4 TB/s, backward 105 us = 5.0 TB/s; 127 363 x 96 fp16 with one rms norm: 20 us = 4.9 TB/s.
#include "common.cuh"
#include "elem.cuh"
#include "ptx.cuh"

namespace sb {

static_assert(sizeof(spira_b200_norm_desc) == 248, "spira_b200_norm_desc layout");

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
  int n, x_stride, block_stride, gate_stride, dstream_stride, dnormed_stride;      // (element strides below 2^31: one wide multiply per row)
  int channels, layer, pre, post, gate_kind, params_f32;
  float residual_scale, block_scale, eps, inv_channels;
};

// Arithmetic on V neighbouring channels, two at a time where V is even (packed fp32 instructions: half the issue slots).
__device__ __forceinline__ void fma2(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float &d0, float &d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add2(float &d0, float &d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
template <int V>
struct Ops {
  typedef float A[V];
  // d = a * b + c
  static __device__ __forceinline__ void fma(A &d, const A &a, const A &b, const A &c) {
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 2) fma2(d[e], d[e + 1], a[e], a[e + 1], b[e], b[e + 1], c[e], c[e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = fmaf(a[e], b[e], c[e]);
    }
  }
  // d = a * s + c
  static __device__ __forceinline__ void fma(A &d, const A &a, float s, const A &c) {
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 2) fma2(d[e], d[e + 1], a[e], a[e + 1], s, s, c[e], c[e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = fmaf(a[e], s, c[e]);
    }
  }
  // d = a * s + t
  static __device__ __forceinline__ void fma(A &d, const A &a, float s, float t) {
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 2) fma2(d[e], d[e + 1], a[e], a[e + 1], s, s, t, t);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = fmaf(a[e], s, t);
    }
  }
  static __device__ __forceinline__ void mul(A &d, const A &a, const A &b) {
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 2) mul2(d[e], d[e + 1], a[e], a[e + 1], b[e], b[e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = a[e] * b[e];
    }
  }
  static __device__ __forceinline__ void mul(A &d, const A &a, float s) {
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 2) mul2(d[e], d[e + 1], a[e], a[e + 1], s, s);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = a[e] * s;
    }
  }
  static __device__ __forceinline__ void add(A &d, const A &a, const A &b) {
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 2) add2(d[e], d[e + 1], a[e], a[e + 1], b[e], b[e + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = a[e] + b[e];
    }
  }
  static __device__ __forceinline__ void add(A &d, const A &a, float t) {
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 2) add2(d[e], d[e + 1], a[e], a[e + 1], t, t);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = a[e] + t;
    }
  }
  static __device__ __forceinline__ float sum(const A &a) {
    if constexpr (V == 8) {
      float t[4];
      add2(t[0], t[1], a[0], a[1], a[2], a[3]);
      add2(t[2], t[3], a[4], a[5], a[6], a[7]);
      add2(t[0], t[1], t[0], t[1], t[2], t[3]);
      return t[0] + t[1];
    } else if constexpr (V == 4) {
      float t[2];
      add2(t[0], t[1], a[0], a[1], a[2], a[3]);
      return t[0] + t[1];
    } else {
      float t = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) t += a[e];
      return t;
    }
  }
  static __device__ __forceinline__ float dot(const A &a, const A &b) {
    if constexpr (V == 8 || V == 4) {
      float t[2];
      mul2(t[0], t[1], a[0], a[1], b[0], b[1]);
#pragma unroll
      for (int e = 2; e < V; e += 2) fma2(t[0], t[1], a[e], a[e + 1], b[e], b[e + 1], t[0], t[1]);
      return t[0] + t[1];
    } else {
      float t = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) t = fmaf(a[e], b[e], t);
      return t;
    }
  }
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

// v[r] = w * v[r] + b with what there is of the two parameters, for R rows.  BOTH: they usually come together (layer norms),
// which is then one instruction per pair (127 363 x 256 bf16 forward 63 -> 62, backward 110 -> 107 us); asking for the pair
// costs rms norms, which rarely have a bias, 20 registers (127 363 x 96 fp16 21.4 -> 23.4 us, held to three CTAs per SM 22.0).
template <typename T, int V, int R, bool BOTH>
__device__ __forceinline__ void affine(const void *w, const void *b, int f32, int c, float (&v)[R][V]) {
  float q[V], t[V];
  if (BOTH && w && b) {
    load_param<T, V>(w, f32, c, q);
    load_param<T, V>(b, f32, c, t);
#pragma unroll
    for (int r = 0; r < R; ++r) Ops<V>::fma(v[r], v[r], q, t);
    return;
  }
  if (w) {
    load_param<T, V>(w, f32, c, q);
#pragma unroll
    for (int r = 0; r < R; ++r) Ops<V>::mul(v[r], v[r], q);
  }
  if (b) {
    load_param<T, V>(b, f32, c, t);
#pragma unroll
    for (int r = 0; r < R; ++r) Ops<V>::add(v[r], v[r], t);
  }
}

// v becomes (v - mean) / deviation for R rows at once; mean and 1 / deviation are returned.  Pieces outside the row are skipped.
template <int L, int ITEMS, int R, int V, bool LAYER>
__device__ __forceinline__ void normalise(float (&v)[ITEMS][R][V], const bool (&in)[ITEMS], const NormParams &P, float *scratch, float (&mean)[R], float (&dev)[R]) {
  float s[R];
  if (LAYER) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (in[i]) s[r] += Ops<V>::sum(v[i][r]);
    }
    row_sums<L, R>(s, scratch);
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = s[r] * P.inv_channels;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    s[r] = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (LAYER) Ops<V>::add(v[i][r], v[i][r], -mean[r]);
      const float t = Ops<V>::dot(v[i][r], v[i][r]);
      if (in[i]) s[r] += t;
    }
  }
  row_sums<L, R>(s, scratch);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    dev[r] = rsqrtf(fmaf(s[r], P.inv_channels, P.eps));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) Ops<V>::mul(v[i][r], v[i][r], dev[r]);
  }
}

// Threads of a CTA: 256, or the row's if it takes more.
template <int L>
constexpr int kNormThreads = L > 256 ? L : 256;
// The backward pass with two rows per thread: the parameters are read once for both and their sums overlap.  Registers decide:
// 384 threads of 168 for pieces of 8 channels (127 363 x 256 bf16, layer, both sides, gate per element: 111 us; 256 threads
// 136 us, 448 and spilling 149 us; one row at a time and twice 256 threads 125 us), 512 of 128 for pieces of 4
// (127 363 x 128 fp32: 97 us, with 384 threads 103 us).
template <int V, int L, int R>
constexpr int kBackwardThreads = R == 1 ? kNormThreads<L> : V == 4 ? 512 : 384;

// The rows on their way: every thread copies its own 16-byte pieces of the next rows into shared memory (cp.async, past the
// L1, where the parameters stay) and reads them back itself, so no barrier is needed and no register waits for a load.
// A ring of kDepth rounds of `tensors` x PER pieces per thread; no ring (kDepth 0) where pieces are not 16 bytes or MOST
// tensors would take too much room.
template <int THREADS, int PER, int MOST, bool WIDE>
struct Ring {
  static constexpr int kMostStage = THREADS * PER * MOST * 16;
  static constexpr int kDepth = !WIDE ? 0 : kMostStage <= 40 * 1024 ? 3 : kMostStage <= 80 * 1024 ? 2 : 0;
  static constexpr int bytes(int tensors) { return kDepth * THREADS * PER * 16 * tensors; }
  unsigned char *base;      // this thread's first piece
  int stage_bytes;
  __device__ __forceinline__ Ring(unsigned char *smem, int tensors) : base(smem + threadIdx.x * 16), stage_bytes(THREADS * PER * 16 * tensors) {}
  __device__ __forceinline__ unsigned char *piece(int stage, int i) const { return base + stage * stage_bytes + i * (THREADS * 16); }
  __device__ __forceinline__ void copy(int stage, int i, const void *src) const { ptx::cp_async_16(ptx::smem_u32(piece(stage, i)), src, 16); }
  static __device__ __forceinline__ void commit() { ptx::cp_async_commit(); }
  static __device__ __forceinline__ void wait() { ptx::cp_async_wait<kDepth == 0 ? 0 : kDepth - 1>(); }
};
// Tensors whose rows go through the ring, in the kernels' order.
__host__ __device__ __forceinline__ int forward_tensors(const NormParams &P) { return P.gate_kind == kGateFull ? 3 : P.block ? 2 : 1; }
__host__ __device__ __forceinline__ int backward_tensors(const NormParams &P) { return P.gate_kind == kGateFull ? 5 : P.dstream ? 4 : P.block ? 3 : 2; }

// L threads per row, each with ITEMS pieces of V neighbouring channels, L pieces apart, and R rows at once.  What limits
// these kernels is not memory alone but instructions and the latency of a row's chain (load, row sum, row sum, store):
// loads run rounds ahead, options are tested per row and never per element, conversions and arithmetic work on pairs, two rows share the parameter
// loads and overlap their sums.  Loads are clamped into the tensor instead of guarded; only stores and sums ask whether a
// row or a piece exists.  Pieces of 8 are held to 80 registers (no spills), so that three CTAs fit on an SM.
template <typename T, int V, int L, int ITEMS, int R, bool LAYER>
__global__ void __launch_bounds__(kNormThreads<L>, V == 8 && L <= 32 && ITEMS == 1 ? 3 : 1) norm_forward_kernel(const __grid_constant__ NormParams P) {
  __shared__ float scratch[64];
  pdl_trigger();
  pdl_wait();
  const int g = threadIdx.x % L;
  constexpr int kRows = kNormThreads<L> / L;
  const int rounds = (P.n + kRows * R - 1) / (kRows * R);
  bool in[ITEMS];
  int col[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    in[i] = (i * L + g) * V < P.channels;
    col[i] = in[i] ? (i * L + g) * V : 0;
  }
  extern __shared__ __align__(16) unsigned char norm_ring[];
  typedef Ring<kNormThreads<L>, ITEMS * R, 3, V * sizeof(T) == 16> Rows;
  const Rows ring(norm_ring, forward_tensors(P));
  constexpr int kDepth = Rows::kDepth;
  auto source = [&](int which, int64_t row, int c) -> const T * {
    if (which == 0) return static_cast<const T *>(P.x) + row * P.x_stride + c;
    if (which == 1) return static_cast<const T *>(P.block) + row * P.block_stride + c;
    return static_cast<const T *>(P.gate) + row * P.gate_stride + c;
  };
  const bool used[3] = {true, P.block != nullptr, P.gate_kind == kGateFull};
  auto row_of = [&](int b, int r) {
    const int row = (b * kRows + static_cast<int>(threadIdx.x) / L) * R + r;
    return row < P.n ? row : P.n - 1;
  };
  auto fetch = [&](int stage, int b) {
    if (b < rounds)
#pragma unroll
      for (int w = 0; w < 3; ++w)
        if (used[w])
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) ring.copy(stage, (w * R + r) * ITEMS + i, source(w, row_of(b, r), col[i]));
    Rows::commit();
  };
  auto take = [&](int stage, int w, int r, int i, int64_t row) -> Vec<T, V> {
    if constexpr (kDepth > 0) return *reinterpret_cast<const Vec<T, V> *>(ring.piece(stage, (w * R + r) * ITEMS + i));
    else return *reinterpret_cast<const Vec<T, V> *>(source(w, row, col[i]));
  };
  int stage = 0;
  if constexpr (kDepth > 0)
    for (int k = 0; k < kDepth - 1; ++k) fetch(k, blockIdx.x + k * gridDim.x);
  for (int b = blockIdx.x; b < rounds; b += gridDim.x) {
    if constexpr (kDepth > 0) {
      fetch(stage == 0 ? kDepth - 1 : stage - 1, b + (kDepth - 1) * gridDim.x);
      Rows::wait();
    }
    const int row0 = (b * kRows + static_cast<int>(threadIdx.x) / L) * R;
    float x[ITEMS][R][V], p[ITEMS][R][V];
    Vec<T, V> gates[ITEMS][R];
    float row_gate[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row_of(b, r);
      row_gate[r] = P.block_scale;
      if (P.gate_kind == kGateRow) row_gate[r] *= to_f32(static_cast<const T *>(P.gate)[row * P.gate_stride]);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        vec_to_f32<T, V>(take(stage, 0, r, i, row), x[i][r]);
        if (P.block) vec_to_f32<T, V>(take(stage, 1, r, i, row), p[i][r]);
        if (P.gate_kind == kGateFull) gates[i][r] = take(stage, 2, r, i, row);
      }
    }
    if (++stage >= kDepth) stage = 0;
    float block_mean[R] = {}, block_dev[R] = {}, mean[R] = {}, dev[R] = {};
    if (P.block) {
      if (P.post) {
        normalise<L, ITEMS, R, V, LAYER>(p, in, P, scratch, block_mean, block_dev);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) affine<T, V, R, LAYER>(P.post_weight, P.post_bias, P.params_f32, col[i], p[i]);
      }
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (P.gate_kind == kGateChannel) affine<T, V, R, LAYER>(P.gate, nullptr, P.params_f32, col[i], p[i]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (P.gate_kind == kGateFull) {
            float f[V];
            vec_to_f32<T, V>(gates[i][r], f);
            Ops<V>::mul(p[i][r], p[i][r], f);
          }
          Ops<V>::mul(x[i][r], x[i][r], P.residual_scale);
          Ops<V>::fma(x[i][r], p[i][r], row_gate[r], x[i][r]);
          if (in[i] && row0 + r < P.n) store_f32<T, V>(static_cast<T *>(P.stream) + static_cast<int64_t>(row0 + r) * P.channels + col[i], x[i][r]);
        }
      }
    }
    if (P.pre) {
      normalise<L, ITEMS, R, V, LAYER>(x, in, P, scratch, mean, dev);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        affine<T, V, R, LAYER>(P.weight, P.bias, P.params_f32, col[i], x[i]);
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (in[i] && row0 + r < P.n) store_f32<T, V>(static_cast<T *>(P.normed) + static_cast<int64_t>(row0 + r) * P.channels + col[i], x[i][r]);
      }
    }
    if (P.stats && g == 0)
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r < P.n) reinterpret_cast<float4 *>(P.stats)[row0 + r] = make_float4(block_mean[r], block_dev[r], mean[r], dev[r]);
  }
}

template <typename T, int V, int L, int ITEMS, int R, bool LAYER>
__global__ void __launch_bounds__(kBackwardThreads<V, L, R>, L > 32 || ITEMS > 1 || R > 1 ? 1 : 2) norm_backward_kernel(const __grid_constant__ NormParams P) {
  constexpr int kThreads = kBackwardThreads<V, L, R>;
  __shared__ float scratch[64];
  extern __shared__ __align__(16) unsigned char norm_ring[];
  float *column_sums = reinterpret_cast<float *>(norm_ring);      // [kThreads / L][channels], once the rows are through
  pdl_trigger();
  pdl_wait();
  typedef Ops<V> O;
  const int g = threadIdx.x % L;
  constexpr int kRows = kThreads / L, kBoth = LAYER ? 2 : 1;
  const int rounds = (P.n + kRows * R - 1) / (kRows * R);
  const float a = P.block ? P.residual_scale : 1.f, s = P.block_scale;
  const void *post_w = P.post ? P.post_weight : nullptr, *post_b = P.post ? P.post_bias : nullptr;
  bool in[ITEMS];
  int col[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    in[i] = (i * L + g) * V < P.channels;
    col[i] = in[i] ? (i * L + g) * V : 0;
  }
  typedef Ring<kThreads, ITEMS * R, 5, V * sizeof(T) == 16> Rows;
  const Rows ring(norm_ring, backward_tensors(P));
  constexpr int kDepth = Rows::kDepth;
  // 0: x, 1: gradient of the normed rows, 2: block, 3: gradient of the stream, 4: gate
  auto source = [&](int which, int64_t row, int c) -> const T * {
    if (which == 0) return static_cast<const T *>(P.x) + row * P.x_stride + c;
    if (which == 1) return static_cast<const T *>(P.dnormed) + row * P.dnormed_stride + c;
    if (which == 2) return static_cast<const T *>(P.block) + row * P.block_stride + c;
    if (which == 3) return static_cast<const T *>(P.dstream) + row * P.dstream_stride + c;
    return static_cast<const T *>(P.gate) + row * P.gate_stride + c;
  };
  const bool used[5] = {P.pre != 0, P.pre != 0, P.block != nullptr, P.dstream != nullptr, P.gate_kind == kGateFull};
  auto row_of = [&](int b, int r) {
    const int row = (b * kRows + static_cast<int>(threadIdx.x) / L) * R + r;
    return row < P.n ? row : P.n - 1;
  };
  auto fetch = [&](int stage, int b) {
    if (b < rounds)
#pragma unroll
      for (int w = 0; w < 5; ++w)
        if (used[w])
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) ring.copy(stage, (w * R + r) * ITEMS + i, source(w, row_of(b, r), col[i]));
    Rows::commit();
  };
  auto take = [&](int stage, int w, int r, int i, int64_t row) -> Vec<T, V> {
    if constexpr (kDepth > 0) return *reinterpret_cast<const Vec<T, V> *>(ring.piece(stage, (w * R + r) * ITEMS + i));
    else return *reinterpret_cast<const Vec<T, V> *>(source(w, row, col[i]));
  };
  int stage = 0;
  if constexpr (kDepth > 0)
    for (int k = 0; k < kDepth - 1; ++k) fetch(k, blockIdx.x + k * gridDim.x);
  float sum[kSums][ITEMS][V] = {};
  for (int b = blockIdx.x; b < rounds; b += gridDim.x) {
    if constexpr (kDepth > 0) {
      fetch(stage == 0 ? kDepth - 1 : stage - 1, b + (kDepth - 1) * gridDim.x);
      Rows::wait();
    }
    const int row0 = (b * kRows + static_cast<int>(threadIdx.x) / L) * R;
    bool live[R];
    int64_t row[R];
    float4 st[R];
    // hat: x, then the stream's normalised value; bh: the block's normalised value (or the block); q: its affine form times
    // the gate; d: gradient of the stream
    float hat[ITEMS][R][V], bh[ITEMS][R][V], d[ITEMS][R][V], u[ITEMS][R][V], q[ITEMS][R][V];
    Vec<T, V> gates[ITEMS][R];
    float row_gate[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      live[r] = row0 + r < P.n;
      row[r] = row_of(b, r);
      st[r] = reinterpret_cast<const float4 *>(P.stats)[row[r]];
      row_gate[r] = P.gate_kind == kGateRow ? to_f32(static_cast<const T *>(P.gate)[row[r] * P.gate_stride]) : 1.f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (P.pre) {
          vec_to_f32<T, V>(take(stage, 0, r, i, row[r]), hat[i][r]);
          vec_to_f32<T, V>(take(stage, 1, r, i, row[r]), u[i][r]);
        }
        if (P.block) vec_to_f32<T, V>(take(stage, 2, r, i, row[r]), bh[i][r]);
        if (P.dstream) {
          vec_to_f32<T, V>(take(stage, 3, r, i, row[r]), d[i][r]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) d[i][r][e] = 0.f;
        }
        if (P.gate_kind == kGateFull) gates[i][r] = take(stage, 4, r, i, row[r]);
      }
    }
    if (++stage >= kDepth) stage = 0;
    auto load_gate = [&](int i, int r, float (&f)[V]) {
      if (P.gate_kind == kGateChannel) load_param<T, V>(P.gate, P.params_f32, col[i], f);
      else vec_to_f32<T, V>(gates[i][r], f);
    };
    float sums[kBoth * R];      // [R], then [R] with kLayer
    if (P.block) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (P.post) O::fma(bh[i][r], bh[i][r], st[r].y, LAYER ? -st[r].x * st[r].y : 0.f);
#pragma unroll
          for (int e = 0; e < V; ++e) q[i][r][e] = bh[i][r][e];
        }
        affine<T, V, R, LAYER>(post_w, post_b, P.params_f32, col[i], q[i]);
      }
    }
    if (P.pre) {
#pragma unroll
      for (int m = 0; m < kBoth * R; ++m) sums[m] = 0.f;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (P.block) {
            O::mul(hat[i][r], hat[i][r], a);
            if (P.gate_kind == kGateNone || P.gate_kind == kGateRow) {
              O::fma(hat[i][r], q[i][r], s * row_gate[r], hat[i][r]);
            } else {
              float f[V];
              load_gate(i, r, f);
              O::mul(f, f, q[i][r]);
              O::fma(hat[i][r], f, s, hat[i][r]);
            }
          }
          O::fma(hat[i][r], hat[i][r], st[r].w, LAYER ? -st[r].z * st[r].w : 0.f);
          if (live[r]) {                                          // (a row that does not exist adds nothing to the column sums)
            O::fma(sum[0][i], u[i][r], hat[i][r], sum[0][i]);
            O::add(sum[1][i], sum[1][i], u[i][r]);
          }
        }
        affine<T, V, R, LAYER>(P.weight, nullptr, P.params_f32, col[i], u[i]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float t0 = O::dot(u[i][r], hat[i][r]), t1 = LAYER ? O::sum(u[i][r]) : 0.f;
          if (in[i]) {
            sums[r] += t0;
            if (LAYER) sums[(kBoth - 1) * R + r] += t1;
          }
        }
      }
      row_sums<L, kBoth * R>(sums, scratch);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float m0 = -sums[r] * P.inv_channels * st[r].w, m1 = LAYER ? -sums[(kBoth - 1) * R + r] * P.inv_channels * st[r].w : 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          if (LAYER) O::add(d[i][r], d[i][r], m1);
          O::fma(d[i][r], u[i][r], st[r].w, d[i][r]);
          O::fma(d[i][r], hat[i][r], m0, d[i][r]);
        }
      }
    }
    if (P.dx)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          float o[V];
          O::mul(o, d[i][r], a);
          if (live[r] && in[i]) store_f32<T, V>(static_cast<T *>(P.dx) + row[r] * P.channels + col[i], o);
        }
    if (P.block) {
#pragma unroll
      for (int m = 0; m < kBoth * R; ++m) sums[m] = 0.f;
      float gate_sum[R] = {};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          O::mul(d[i][r], d[i][r], s);
          if (P.gate_kind != kGateNone) {
            O::mul(q[i][r], q[i][r], d[i][r]);                  // gradient of the gate
            if (P.gate_kind == kGateRow) {
              const float t = O::sum(q[i][r]);
              if (in[i]) gate_sum[r] += t;
              O::mul(d[i][r], d[i][r], row_gate[r]);
            } else {
              if (P.gate_kind == kGateChannel && live[r]) O::add(sum[4][i], sum[4][i], q[i][r]);
              if (P.gate_kind == kGateFull && P.dgate && live[r] && in[i])
                store_f32<T, V>(static_cast<T *>(P.dgate) + row[r] * P.channels + col[i], q[i][r]);
              float f[V];
              load_gate(i, r, f);
              O::mul(d[i][r], d[i][r], f);
            }
          }
        }
        if (P.post) {
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (live[r]) {
              O::fma(sum[2][i], d[i][r], bh[i][r], sum[2][i]);
              O::add(sum[3][i], sum[3][i], d[i][r]);
            }
          affine<T, V, R, LAYER>(post_w, nullptr, P.params_f32, col[i], d[i]);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float t0 = O::dot(d[i][r], bh[i][r]), t1 = LAYER ? O::sum(d[i][r]) : 0.f;
            if (in[i]) {
              sums[r] += t0;
              if (LAYER) sums[(kBoth - 1) * R + r] += t1;
            }
          }
        }
      }
      if (P.gate_kind == kGateRow && P.dgate) {
        row_sums<L, R>(gate_sum, scratch);
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (live[r] && g == 0) static_cast<T *>(P.dgate)[row[r]] = from_f32<T>(gate_sum[r]);
      }
      if (P.dblock) {
        if (P.post) {
          row_sums<L, kBoth * R>(sums, scratch);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float m0 = -sums[r] * P.inv_channels, m1 = LAYER ? -sums[(kBoth - 1) * R + r] * P.inv_channels : 0.f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
              if (LAYER) O::add(d[i][r], d[i][r], m1);
              O::fma(d[i][r], bh[i][r], m0, d[i][r]);
              O::mul(d[i][r], d[i][r], st[r].y);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < ITEMS; ++i)
            if (live[r] && in[i]) store_f32<T, V>(static_cast<T *>(P.dblock) + row[r] * P.channels + col[i], d[i][r]);
      }
    }
  }
  if (P.partial == nullptr) return;
  if constexpr (kDepth > 0) ptx::cp_async_wait<0>();
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

// CTAs of a kernel that fit on an SM with its shared memory, asked once per kernel and number of tensors (`known`; the answer is
// the same whoever writes it, and a query that failed leaves none).
template <typename K>
static int resident_ctas(K kernel, int threads, int smem, int &known) {
  int n = known;
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) return 1;
    known = n;
  }
  return n;
}

template <typename T, int V, int L, int ITEMS, bool LAYER>
static int launch_norm_kind(const NormParams &P, bool backward, int *ctas, cudaStream_t st) {
  constexpr int kThreads = kNormThreads<L>;
  constexpr int kRows = kThreads / L;
  constexpr bool kWide = V * sizeof(T) == 16;
  if (!backward) {
    constexpr int R = L <= 32 && ITEMS == 1 ? 2 : 1;
    typedef Ring<kThreads, ITEMS * R, 3, kWide> Rows;
    const int tensors = forward_tensors(P), smem = Rows::bytes(tensors);
    const auto kernel = norm_forward_kernel<T, V, L, ITEMS, R, LAYER>;
    const int64_t rounds = div_up(P.n, kRows * R);
    const int rc = allow_smem(kernel, Rows::bytes(3));
    if (rc != SPIRA_B200_OK) return rc;
    static int resident[4] = {0, 0, 0, 0};
    const int64_t cap = static_cast<int64_t>(sm_count()) * resident_ctas(kernel, kThreads, smem, resident[tensors]);
    SB_CHECK_CUDA(launch_operator(kernel, dim3(static_cast<unsigned>(rounds < cap ? rounds : cap)), dim3(kThreads), smem, st, P));
    return SPIRA_B200_OK;
  }
  constexpr int RB = L <= 32 && ITEMS == 1 ? 2 : 1, kBackward = kBackwardThreads<V, L, RB>, kBackwardRows = kBackward / L;
  // (column sums of a CTA reuse the ring: kBackward / L rows of L * ITEMS * V columns)
  constexpr int kColumns = kBackwardRows > 1 ? kBackward * ITEMS * V * 4 : 0;
  typedef Ring<kBackward, ITEMS * RB, 5, kWide> Rows;
  auto need = [](int tensors) { return Rows::bytes(tensors) > kColumns ? Rows::bytes(tensors) : kColumns; };
  const int tensors = backward_tensors(P), smem = need(tensors);
  const auto kernel = norm_backward_kernel<T, V, L, ITEMS, RB, LAYER>;
  const int64_t rounds = div_up(P.n, kBackwardRows * RB);
  const int rc = allow_smem(kernel, need(5));
  if (rc != SPIRA_B200_OK) return rc;
  static int resident[6] = {0, 0, 0, 0, 0, 0};
  const int fit = resident_ctas(kernel, kBackward, smem, resident[tensors]);
  const int64_t cap = static_cast<int64_t>(sm_count()) * (fit < kNormBackwardCtas ? fit : kNormBackwardCtas);
  const int grid = static_cast<int>(rounds < cap ? rounds : cap);
  *ctas = grid;
  SB_CHECK_CUDA(launch_operator(kernel, dim3(grid), dim3(kBackward), smem, st, P));
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
  SB_CHECK_ARG(D->n >= 0 && D->n < (int64_t(1) << 31) - 65536, "%s: n=%lld out of range", what, (long long)D->n);
  SB_CHECK_ARG(D->channels >= 1 && D->channels <= kNormMaxChannels, "%s: channels=%d must be 1 to %d", what, D->channels, kNormMaxChannels);
  SB_CHECK_ARG(D->gate_kind >= kGateNone && D->gate_kind <= kGateFull, "%s: unknown gate %d", what, D->gate_kind);
  SB_CHECK_ARG(D->eps > 0.f, "%s: eps must be positive", what);
  SB_CHECK_ARG(D->x_stride >= 0 && D->block_stride >= 0 && D->gate_stride >= 0 && D->dstream_stride >= 0 && D->dnormed_stride >= 0,
               "%s: negative row stride", what);
  SB_CHECK_ARG((D->x_stride | D->block_stride | D->gate_stride | D->dstream_stride | D->dnormed_stride) < (int64_t(1) << 31),
               "%s: rows more than 2^31 elements apart", what);
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
  P.n = static_cast<int>(D.n); P.x_stride = static_cast<int>(D.x_stride); P.block_stride = static_cast<int>(D.block_stride); P.gate_stride = static_cast<int>(D.gate_stride);
  P.dstream_stride = static_cast<int>(D.dstream_stride); P.dnormed_stride = static_cast<int>(D.dnormed_stride);
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
    SB_CHECK_CUDA(launch_operator(norm_sums_kernel<T>, dim3(static_cast<unsigned>(div_up(D.channels, 32)), kSums), dim3(1024), 0, st, S));
    return SPIRA_B200_OK;
  });
}
