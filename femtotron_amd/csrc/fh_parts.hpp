// Sums over fp32 partial rows, deterministic, in one launch: what the blocks of a
// backward leave of a vector's gradient.
#pragma once

#include "fh_common.hpp"

namespace fh {

// sum_p part[p * ld + c] over p < nparts for the 16 columns c = 16 blockIdx.x + i, in
// threads i < 16 of a block of 256 (of which all call this; cols % 8 == 0 and the
// rows 16-byte aligned).  The threads are 64 row groups x 4 column quads; thread (g,
// q) sums the float4 of rows p = g, g + 64, g + 128, ... in order (eight loads in
// flight), and the 64 group sums of a column are added in group order.  One launch
// instead of a partial pass plus a stage pass measured 1-2 us faster per backward
// call (one launch gap fewer).
__device__ __forceinline__ float sum_parts(const float* __restrict__ part, int64_t ld, int nparts, int cols) {
  constexpr int G = 64, U = 8;
  __shared__ float red[G][17];
  const int q = threadIdx.x & 3, g = threadIdx.x >> 2;
  const int c = blockIdx.x * 16 + q * 4;  // cols % 8 == 0: a quad is wholly in or out
  float4 s = {0.f, 0.f, 0.f, 0.f};
  if (c < cols) {
    auto at = [&](int p) { return *reinterpret_cast<const float4*>(part + p * ld + c); };
    int p = g;
    for (; p + G * (U - 1) < nparts; p += G * U) {
      float4 v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = at(p + G * k);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        s.x += v[k].x; s.y += v[k].y; s.z += v[k].z; s.w += v[k].w;
      }
    }
    for (; p < nparts; p += G) {
      const float4 v = at(p);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  red[g][q * 4 + 0] = s.x;
  red[g][q * 4 + 1] = s.y;
  red[g][q * 4 + 2] = s.z;
  red[g][q * 4 + 3] = s.w;
  __syncthreads();
  float t = 0.f;
  if (threadIdx.x < 16)
    for (int k = 0; k < G; ++k) t += red[k][threadIdx.x];
  return t;
}

}  // namespace fh
