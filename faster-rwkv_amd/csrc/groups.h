// Groups of consecutive elements, in fp32 on the device, at any address that is a multiple of their element's size.
#pragma once

#include "device_utils.h"

namespace frhip {

template <class T>
constexpr int kGroup = 16 / sizeof(T);  // elements of an access of 16 bytes

// Up to V elements at any address of one, the first n of them; 16 bytes an instruction if all are there, as for aligned ones
template <class T, int V>
__device__ __forceinline__ void load_group(float (&v)[V], const T* p, int n) {
  constexpr int P = V < kGroup<T> ? V : kGroup<T>;
  typedef T any __attribute__((ext_vector_type(P), aligned(sizeof(T))));
  static_assert(V % P == 0, "whole pieces");
  if (n >= V) {
#pragma unroll
    for (int q = 0; q < V; q += P) {
      const any t = *reinterpret_cast<const any*>(p + q);
#pragma unroll
      for (int i = 0; i < P; i++) v[q + i] = (float)t[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i < n ? (float)p[i] : 0.f;
  }
}
template <class T, int V>
__device__ __forceinline__ void store_group(T* p, const float (&v)[V], int n) {
  typedef T any __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if (n >= V) {
    any t;
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = (T)v[i];
    *reinterpret_cast<any*>(p) = t;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = (T)v[i];
  }
}

}  // namespace frhip
