// Helpers of the row operators (layer_norm.hip, rope.hip, token_logprobs.hip, route_experts.hip): element types, 16-byte
// accesses at any element alignment, wave-wide reductions, and the host's dispatch over element types.
#pragma once

#include <hip/hip_runtime.h>
#include <c10/core/DeviceGuard.h>

#include "common.h"

namespace acc {

using half_t = _Float16;
template <> __device__ __forceinline__ float to_f<half_t>(half_t x) { return static_cast<float>(x); }
template <> __device__ __forceinline__ half_t from_f<half_t>(float x) { return static_cast<half_t>(x); }

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// N elements in one access from an address that is a multiple of the element size only: global memory takes 16-byte
// accesses at any alignment, so rows of odd width, and views at odd offsets, move as wide as aligned ones.
template <int BYTES> struct RawVec;
template <> struct RawVec<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
template <> struct RawVec<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <> struct RawVec<4> { typedef uint32_t type; };
template <> struct RawVec<2> { typedef uint16_t type; };

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_any(const T* p) {
  typedef typename RawVec<sizeof(T) * N>::type raw;
  typedef raw loose __attribute__((aligned(sizeof(T))));
  return __builtin_bit_cast(Pack<T, N>, static_cast<raw>(*reinterpret_cast<const loose*>(p)));
}

template <typename T, int N>
__device__ __forceinline__ void store_any(T* p, const Pack<T, N>& x) {
  typedef typename RawVec<sizeof(T) * N>::type raw;
  typedef raw loose __attribute__((aligned(sizeof(T))));
  *reinterpret_cast<loose*>(p) = __builtin_bit_cast(raw, x);
}

// The same for chunks wider than 16 bytes (a row operator's fp32 weights beside 16-bit rows).
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_wide(const T* p) {
  if constexpr (sizeof(T) * N <= 16) {
    return load_any<T, N>(p);
  } else {
    struct Halves { Pack<T, N / 2> lo, hi; } h{load_wide<T, N / 2>(p), load_wide<T, N / 2>(p + N / 2)};
    return __builtin_bit_cast(Pack<T, N>, h);
  }
}

// Elements [0, n) of a chunk, n < N: the end of a row whose width is no multiple of N. The rest is zero.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_part(const T* p, int n) {
  Pack<T, N> x;
#pragma unroll
  for (int j = 0; j < N; ++j) x.v[j] = j < n ? p[j] : T(0);
  return x;
}

template <typename T, int N>
__device__ __forceinline__ void store_part(T* p, const Pack<T, N>& x, int n) {
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < n) p[j] = x.v[j];
}

// Reductions over the 64 lanes in registers: two quad permutes, two mirrors within 16 lanes, then exchanges of 16 and 32
// lanes. Every lane ends with the same bits (each step adds the same two numbers on both sides).
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
struct OpSum { static __device__ __forceinline__ float of(float a, float b) { return a + b; } };
struct OpMax { static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); } };

template <typename Op>
__device__ __forceinline__ float wave_reduce(float v) {
  v = Op::of(v, dpp_move<0xB1>(v));   // quad_perm 1,0,3,2
  v = Op::of(v, dpp_move<0x4E>(v));   // quad_perm 2,3,0,1
  v = Op::of(v, dpp_move<0x141>(v));  // row_half_mirror
  v = Op::of(v, dpp_move<0x140>(v));  // row_mirror
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = Op::of(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return Op::of(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The same over THREADS threads that form a block (or over one wave). `slots`: 16 floats of shared memory that no other
// reduction uses between two barriers of the block.
template <typename Op, int THREADS>
__device__ __forceinline__ float row_reduce(float v, float* slots) {
  v = wave_reduce<Op>(v);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slots[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) v = Op::of(v, slots[i]);
  }
  return v;
}

}  // namespace acc

// Runs the statement with `scalar` as the kernels' element type of `dtype`.
#define ACC_FOR_FLOAT_TYPES(dtype, NAME, ...)                                                    \
  do {                                                                                           \
    switch (dtype) {                                                                             \
      case at::kBFloat16: { using scalar = acc::bf16_t; __VA_ARGS__; break; }                    \
      case at::kHalf: { using scalar = acc::half_t; __VA_ARGS__; break; }                        \
      case at::kFloat: { using scalar = float; __VA_ARGS__; break; }                             \
      default: TORCH_CHECK(false, NAME, ": bf16, fp16 or fp32 expected, got ", dtype);           \
    }                                                                                            \
  } while (0)
