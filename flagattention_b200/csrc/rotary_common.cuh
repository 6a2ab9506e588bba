// What the kernels that rotate queries and keys share: eight 16-bit elements to and from fp32, and the two layouts of a
// rotation pair.
#pragma once

#include "common.cuh"

namespace fa {

__device__ __forceinline__ void load8(float (&dst)[8], const float *src) {
  const float4 a = *reinterpret_cast<const float4 *>(src);
  const float4 b = *reinterpret_cast<const float4 *>(src + 4);
  dst[0] = a.x, dst[1] = a.y, dst[2] = a.z, dst[3] = a.w;
  dst[4] = b.x, dst[5] = b.y, dst[6] = b.z, dst[7] = b.w;
}

template <typename T>
__device__ __forceinline__ void unpack8(float (&dst)[8], const uint4 &u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::unpack(w[i]);
    dst[2 * i] = f.x, dst[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint4 u;
  u.x = Elem<T>::pack(v[0], v[1]);
  u.y = Elem<T>::pack(v[2], v[3]);
  u.z = Elem<T>::pack(v[4], v[5]);
  u.w = Elem<T>::pack(v[6], v[7]);
  return u;
}

// a[i], b[i] are the two members of pair i in the half-split layout; in the interleaved layout
// the sixteen values are a[0..7] = elements 0..7 and b[0..7] = elements 8..15 of the thread's run.
template <bool INTERLEAVED>
__device__ __forceinline__ void to_pairs(float (&lo)[8], float (&hi)[8], const float (&a)[8],
                                         const float (&b)[8]) {
  if (INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = a[2 * i], hi[i] = a[2 * i + 1];
      lo[4 + i] = b[2 * i], hi[4 + i] = b[2 * i + 1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = a[i], hi[i] = b[i];
  }
}

template <bool INTERLEAVED>
__device__ __forceinline__ void from_pairs(float (&a)[8], float (&b)[8], const float (&lo)[8],
                                           const float (&hi)[8]) {
  if (INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[2 * i] = lo[i], a[2 * i + 1] = hi[i];
      b[2 * i] = lo[4 + i], b[2 * i + 1] = hi[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = lo[i], b[i] = hi[i];
  }
}

}  // namespace fa
