// Element types of the row-wise operators (fp16, bf16, fp32): conversion, 16-byte vectors, dispatch on the type code.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"

namespace sb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements as one aligned access of N * sizeof(T) bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void vec_to_f32(const Vec<T, N> &r, float (&f)[N]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value && N % 2 == 0) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&r);      // a bf16 is the upper half of its fp32
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      f[i] = __uint_as_float(w[i / 2] << 16);
      f[i + 1] = __uint_as_float(w[i / 2] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32(r.v[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T *p, float (&f)[N]) {
  vec_to_f32<T, N>(*reinterpret_cast<const Vec<T, N> *>(p), f);
}
template <typename T, int N>
__device__ __forceinline__ void store_f32(T *p, const float (&f)[N]) {
  Vec<T, N> r;
  if constexpr (std::is_same<T, __half>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<__half2 *>(&r.v[i]) = __floats2half2_rn(f[i], f[i + 1]);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<__nv_bfloat162 *>(&r.v[i]) = __floats2bfloat162_rn(f[i], f[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(f[i]);
  }
  *reinterpret_cast<Vec<T, N> *>(p) = r;
}

// Allows a kernel `most` bytes of dynamic shared memory (48 KB with its static part need no permission).  The limit belongs to
// the kernel on the current device and not to the call, so `most` is what the largest call of the kernel takes, whatever
// this one needs: a call that set its own size could lower the limit between another thread's setting and its launch.
template <typename K>
inline int allow_smem(K kernel, size_t most) {
  if (most > 40 * 1024) SB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
  return SPIRA_B200_OK;
}

// Kernels of the expert and norm operators launched by this process (how many a call takes depends on its sizes).
void count_operator_launch();
template <typename... KArgs, typename... Args>
inline cudaError_t launch_operator(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args &&...args) {
  const cudaError_t e = launch_dependent(kernel, grid, block, smem, stream, static_cast<Args &&>(args)...);
  if (e == cudaSuccess) count_operator_launch();
  return e;
}

inline int elem_size(int dtype) { return dtype == SPIRA_B200_F32 ? 4 : 2; }

// Runs BODY with T = the element type of the code.
#define SB_DISPATCH_ELEM(dtype, T, ...)                              \
  [&]() -> int {                                                     \
    if ((dtype) == SPIRA_B200_F16) { using T = __half; __VA_ARGS__ } \
    if ((dtype) == SPIRA_B200_BF16) { using T = __nv_bfloat16; __VA_ARGS__ } \
    using T = float; __VA_ARGS__                                     \
  }()

}  // namespace sb
