// Rows of f32, bf16 or f16 in device memory, four columns at a time.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rtg {

// Columns c4 .. c4 + 3 of a row of n, those from n on 0. vec (the same for all
// threads): n % 4 == 0 and the four are aligned to their size.
template <class T>
__device__ __forceinline__ float4 load4(const T* row, int c4, int n, bool vec) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  if (vec) {
    if (c4 >= n) return make_float4(0.f, 0.f, 0.f, 0.f);
    const T4 v = *reinterpret_cast<const T4*>(row + c4);
    return make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
  }
  float r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = c4 + e < n ? (float)row[c4 + e] : 0.f;
  return make_float4(r[0], r[1], r[2], r[3]);
}
template <class T>
__device__ __forceinline__ void store1(T* p, float x) {
  *p = (T)x;  // to nearest even
}
template <class T>
__device__ __forceinline__ void store4(T* row, int c4, int n, const float4& x, bool vec) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  if (vec) {
    if (c4 >= n) return;
    T4 v;
    v[0] = (T)x.x;
    v[1] = (T)x.y;
    v[2] = (T)x.z;
    v[3] = (T)x.w;
    *reinterpret_cast<T4*>(row + c4) = v;
    return;
  }
  const float r[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c4 + e < n) row[c4 + e] = (T)r[e];
}

}  // namespace rtg
