// Helpers of the row operators (layer_norm.hip, rope.hip, token_logprobs.hip, route_experts.hip): element types, 16-byte
// accesses at any element alignment, wave-wide reductions, and the host's dispatch over element types.
#pragma once

#include <hip/hip_runtime.h>
#include <c10/core/DeviceGuard.h>
#include <type_traits>

#include "common.h"

namespace acc {

using half_t = _Float16;
template <> __device__ __forceinline__ float to_f<half_t>(half_t x) { return static_cast<float>(x); }
template <> __device__ __forceinline__ half_t from_f<half_t>(float x) { return static_cast<half_t>(x); }

// N elements as they lie in memory, two 16-bit ones to a register: arrays of 16-bit values end up one to a register.
template <typename T, int N>
struct Pack {
  static constexpr int kWords = sizeof(T) * N < 4 ? 1 : sizeof(T) * N / 4;
  uint32_t u[kWords];

  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(u[j]);
    } else {
      const uint32_t w = u[j / 2];
      if constexpr (std::is_same<T, half_t>::value) return to_f<T>(__builtin_bit_cast(half_t, (uint16_t)(j & 1 ? w >> 16 : w)));
      else return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
    }
  }
  static __device__ __forceinline__ Pack of(const float (&f)[N]) {
    Pack p;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < N; ++j) p.u[j] = __float_as_uint(f[j]);
    } else if constexpr (N == 1) {
      p.u[0] = __builtin_bit_cast(uint16_t, from_f<T>(f[0]));
    } else {
      using hw = typename std::conditional<std::is_same<T, half_t>::value, half_t, __bf16>::type;
      typedef hw pair __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int j = 0; j < N; j += 2) p.u[j / 2] = __builtin_bit_cast(uint32_t, pair{static_cast<hw>(f[j]), static_cast<hw>(f[j + 1])});
    }
    return p;
  }
  // elements [i, i + G) from another pack; they were zero
  template <int G>
  __device__ __forceinline__ void put(int i, const Pack<T, G>& x) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < G; ++j) u[i + j] = x.u[j];
    } else if constexpr (G == 1) {
      u[i / 2] |= x.u[0] << (16 * (i & 1));
    } else {
#pragma unroll
      for (int j = 0; j < G / 2; ++j) u[i / 2 + j] = x.u[j];
    }
  }
  static __device__ __forceinline__ Pack zero() {
    Pack p;
#pragma unroll
    for (int i = 0; i < kWords; ++i) p.u[i] = 0;
    return p;
  }
};

// N elements from an address that is a multiple of the element size only: global memory takes 16-byte accesses at any
// alignment, so rows of odd width, and views at odd offsets, move as wide as aligned ones.
template <int BYTES> struct RawVec;
template <> struct RawVec<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
template <> struct RawVec<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <> struct RawVec<4> { typedef uint32_t type; };
template <> struct RawVec<2> { typedef uint16_t type; };

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_any(const T* p) {
  constexpr int bytes = sizeof(T) * N;
  if constexpr (bytes > 16) {  // fp32 parameters beside 16-bit rows
    const Pack<T, N / 2> lo = load_any<T, N / 2>(p), hi = load_any<T, N / 2>(p + N / 2);
    Pack<T, N> x;
#pragma unroll
    for (int i = 0; i < Pack<T, N / 2>::kWords; ++i) {
      x.u[i] = lo.u[i];
      x.u[Pack<T, N / 2>::kWords + i] = hi.u[i];
    }
    return x;
  } else {
    typedef typename RawVec<bytes>::type raw;
    typedef raw loose __attribute__((aligned(sizeof(T))));
    const raw r = *reinterpret_cast<const loose*>(p);
    if constexpr (bytes == 2) return Pack<T, N>{{r}};
    else return __builtin_bit_cast(Pack<T, N>, r);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_any(T* p, const Pack<T, N>& x) {
  constexpr int bytes = sizeof(T) * N;
  typedef typename RawVec<bytes>::type raw;
  typedef raw loose __attribute__((aligned(sizeof(T))));
  if constexpr (bytes == 2) *reinterpret_cast<loose*>(p) = (uint16_t)x.u[0];
  else *reinterpret_cast<loose*>(p) = __builtin_bit_cast(raw, x);
}

// Elements [0, n) of a chunk, n < N, one by one; the rest is zero.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_part(const T* p, int n) {
  Pack<T, N> x = Pack<T, N>::zero();
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < n) {
      if constexpr (sizeof(T) == 4) x.u[j] = reinterpret_cast<const uint32_t*>(p)[j];
      else x.u[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[j] << (16 * (j & 1));
    }
  return x;
}

// Elements [s, N) of x moved to its front, zero behind them.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> drop_front(Pack<T, N> x, int s) {
  constexpr int words = Pack<T, N>::kWords;
  int by = s;
  if constexpr (sizeof(T) == 2) {
    by = s >> 1;
    if (s & 1) {
#pragma unroll
      for (int i = 0; i < words; ++i) x.u[i] = (x.u[i] >> 16) | (i + 1 < words ? x.u[i + 1] << 16 : 0);
    }
  }
#pragma unroll
  for (int step = 1; step < words; step <<= 1)
    if (by & step) {
#pragma unroll
      for (int i = 0; i < words; ++i) x.u[i] = i + step < words ? x.u[i + step] : 0;
    }
  return x;
}

// load_part at the end of a row, with `before` elements of the row ahead of p: one access that ends with the row and a shift,
// where the row is that long. (Single loads cost the latency of memory each, all of them at once eight addresses.)
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_tail(const T* p, int n, int before) {
  if (n <= 0) return Pack<T, N>::zero();
  if (before >= N - n) return drop_front<T, N>(load_any<T, N>(p - (N - n)), N - n);
  return load_part<T, N>(p, n);
}

template <typename T, int N>
__device__ __forceinline__ void store_part(T* p, const Pack<T, N>& x, int n) {
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < n) {
      if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[j] = x.u[j];
      else reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)(x.u[j / 2] >> (16 * (j & 1)));
    }
}

// Reductions over L lanes (an aligned power of two, 8 to 64) in registers: two quad permutes, mirrors within 8 and 16 lanes, then
// exchanges of 16 and 32 lanes. Every lane ends with the same bits (each step joins the same two values on both sides).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_move(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int L, typename Op>
__device__ __forceinline__ uint32_t lanes_reduce_u32(uint32_t v) {
  static_assert(L == 8 || L == 16 || L == 32 || L == 64, "lanes");
  v = Op::of(v, dpp_move<0xB1>(v));   // quad_perm 1,0,3,2
  v = Op::of(v, dpp_move<0x4E>(v));   // quad_perm 2,3,0,1
  v = Op::of(v, dpp_move<0x141>(v));  // row_half_mirror
  if constexpr (L >= 16) v = Op::of(v, dpp_move<0x140>(v));  // row_mirror
  if constexpr (L >= 32) {
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = Op::of(a[0], a[1]);
  }
  if constexpr (L >= 64) {
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = Op::of(b[0], b[1]);
  }
  return v;
}
struct OpSum {
  static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct OpMax {
  static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
struct OpMaxU32 { static __device__ __forceinline__ uint32_t of(uint32_t a, uint32_t b) { return a > b ? a : b; } };

template <int L, typename Op>
__device__ __forceinline__ float lanes_reduce(float v) { return __uint_as_float(lanes_reduce_u32<L, Op>(__float_as_uint(v))); }
template <typename Op>
__device__ __forceinline__ float wave_reduce(float v) { return lanes_reduce<64, Op>(v); }
template <int L>
__device__ __forceinline__ uint32_t lanes_max_u32(uint32_t v) { return lanes_reduce_u32<L, OpMaxU32>(v); }

// The same over THREADS threads: lanes of a wave, or the threads of a block. `slots`: 16 floats of shared memory that no other
// reduction uses between two barriers of the block.
template <typename Op, int THREADS>
__device__ __forceinline__ float row_reduce(float v, float* slots) {
  v = lanes_reduce<(THREADS < 64 ? THREADS : 64), Op>(v);
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
