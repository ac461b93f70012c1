// Rows of any element type, width and alignment as 16-byte pieces: what the kernels that go over whole rows
// (block norms, log probabilities) share.
//
// A piece is read and written as one 16-byte access at the element type's own alignment: global memory takes
// it at any address, and an aligned piece costs what an aligned access costs.  So one kernel serves odd widths
// and odd row strides; only the elements behind the last whole piece of a row move one by one.
#pragma once

#include "ccq_tile.h"

namespace ccq {

typedef _Float16 f16;

template <typename T>
struct Piece {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec any __attribute__((aligned(sizeof(T))));  // the same at the element's alignment
};

// elements c .. c + N - 1 of a row of D, zeros past its end
template <typename T>
__device__ __forceinline__ typename Piece<T>::vec load_piece(const T* row, int c, int D) {
  constexpr int N = Piece<T>::N;
  if (c + N <= D) return *gmem((const typename Piece<T>::any*)(row + c));
  typename Piece<T>::vec v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = c + i < D ? *gmem(row + c + i) : (T)0.f;
  return v;
}

template <typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int D, const typename Piece<T>::vec& v) {
  constexpr int N = Piece<T>::N;
  if (c + N <= D) {
    *gmem((typename Piece<T>::any*)(row + c)) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (c + i < D) *gmem(row + c + i) = v[i];
}

// The same for a row's last use, and for one that is not read soon: the caches keep what is.
template <typename T>
__device__ __forceinline__ typename Piece<T>::vec load_last(const T* row, int c, int D) {
  if (c + Piece<T>::N <= D) return __builtin_nontemporal_load(gmem((const typename Piece<T>::any*)(row + c)));
  return load_piece(row, c, D);
}
template <typename T>
__device__ __forceinline__ void store_past(T* row, int c, int D, const typename Piece<T>::vec& v) {
  typedef typename Piece<T>::any any;
  if (c + Piece<T>::N <= D) __builtin_nontemporal_store((any)v, gmem((any*)(row + c)));
  else store_piece(row, c, D, v);
}

// sum over groups of L consecutive lanes (L a power of two <= 64)
__device__ __forceinline__ float lanes_sum(float x, int L) {
  for (int o = L >> 1; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

}  // namespace ccq
