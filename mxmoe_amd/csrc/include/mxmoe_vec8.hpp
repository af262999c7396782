// Pieces of eight row elements for the kernels that stream whole rows in any of the three float types: loads and stores of one piece, sums over
// a wave and over a workgroup.
//
// A piece of 16-bit elements is one 16-byte access, of fp32 two.  The pointers carry the alignment of one element only: global memory takes
// 16-byte accesses at any element's address, so views, odd row lengths and row strides need no second form of a kernel; what a row length that is no
// multiple of eight costs is the last piece, which goes element by element.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mxmoe {

typedef float f8 __attribute__((ext_vector_type(8)));

// float types of the C entry points (as the routing's logits_dtype)
enum FloatType { kF16 = 0, kF32 = 1, kBF16 = 2 };
inline size_t float_bytes(int type) { return type == kF32 ? 4 : 2; }

template <typename T>
struct Piece;  // eight elements of T as they are in memory

template <>
struct Piece<_Float16> {
  typedef _Float16 raw __attribute__((ext_vector_type(8)));
  typedef raw mem __attribute__((aligned(2)));
  static __device__ __forceinline__ f8 widen(raw v) { return __builtin_convertvector(v, f8); }
  static __device__ __forceinline__ raw narrow(f8 v) { return __builtin_convertvector(v, raw); }
};
template <>
struct Piece<__bf16> {
  typedef __bf16 raw __attribute__((ext_vector_type(8)));
  typedef raw mem __attribute__((aligned(2)));
  static __device__ __forceinline__ f8 widen(raw v) { return __builtin_convertvector(v, f8); }
  static __device__ __forceinline__ raw narrow(f8 v) { return __builtin_convertvector(v, raw); }
};
template <>
struct Piece<float> {
  typedef f8 raw;
  typedef raw mem __attribute__((aligned(4)));
  static __device__ __forceinline__ f8 widen(raw v) { return v; }
  static __device__ __forceinline__ raw narrow(f8 v) { return v; }
};

// elements 8 c .. 8 c + 7 of a row of K elements, zeros past its end
template <typename T>
__device__ __forceinline__ typename Piece<T>::raw load_piece(const T* row, int c, int K) {
  typename Piece<T>::raw v{};
  if (8 * c + 8 <= K) {
    v = *reinterpret_cast<const typename Piece<T>::mem*>(row + 8 * c);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * c + i < K) v[i] = row[8 * c + i];
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int K, typename Piece<T>::raw v) {
  if (8 * c + 8 <= K) {
    *reinterpret_cast<typename Piece<T>::mem*>(row + 8 * c) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * c + i < K) row[8 * c + i] = v[i];
  }
}
// the same of a vector whose type is known at run time only (norm weights: read once per workgroup, or from a cache)
__device__ __forceinline__ f8 load_piece_of(int type, const void* row, int c, int K) {
  if (type == kF32) return load_piece(reinterpret_cast<const float*>(row), c, K);
  if (type == kF16) return Piece<_Float16>::widen(load_piece(reinterpret_cast<const _Float16*>(row), c, K));
  return Piece<__bf16>::widen(load_piece(reinterpret_cast<const __bf16*>(row), c, K));
}
__device__ __forceinline__ float load_of(int type, const void* p, long i) {
  if (type == kF32) return reinterpret_cast<const float*>(p)[i];
  if (type == kF16) return (float)reinterpret_cast<const _Float16*>(p)[i];
  return (float)reinterpret_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void store_of(int type, void* p, long i, float v) {
  if (type == kF32) reinterpret_cast<float*>(p)[i] = v;
  else if (type == kF16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
  else reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
}

// Sum over the wave, in every lane: lanes of a row of 16 by shifts, rows by the broadcast of their last lanes; the vector ALU alone (a shuffle is
// a round trip through LDS).  All 64 lanes must be active.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = dpp_add<0x111, 0xF>(v);
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);
  v = dpp_add<0x143, 0xC>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sums of N values each over the NT threads of a workgroup, in every thread.  One barrier: callers that sum again pass the other half of
// their LDS (float [2][N * NT / 64]) in turn, so that no wave overwrites what another still reads.
template <int NT, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* lds) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (NT > 64) {
    constexpr int W = NT / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[i * W + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = lds[i * W];
#pragma unroll
      for (int w = 1; w < W; ++w) s += lds[i * W + w];
      v[i] = s;
    }
  }
}

}  // namespace mxmoe
