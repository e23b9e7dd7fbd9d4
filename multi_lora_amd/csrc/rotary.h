// Rotary tables as the paged writes read them.
#pragma once

#include "loads.h"

namespace mlora {

// A chunk of 8 table values at element e, as fp32.
template <class T, bool AL>
__device__ __forceinline__ void rot_chunk(const void* p, int64_t e, bool f32, float* f) {
  if (f32) {
    const float* t = static_cast<const float*>(p) + e;
    if constexpr (AL) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(t), hi = *reinterpret_cast<const f32x4*>(t + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = lo[i], f[4 + i] = hi[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = t[i];
    }
  } else {
    const u32x4 v = load_row_chunk<T, AL>(static_cast<const typename T::raw_t*>(p), static_cast<int>(e), 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = chunk_elem<T>(v, i);
  }
}

}  // namespace mlora
