// Sums over a step's requests, in a block's LDS.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace htree {

// Exclusive sums over the requests in `dst[0 .. B]`, of f(b), saturated at
// `most`.  All 256 threads; `red` holds the waves' sums.
template <typename F>
__device__ __forceinline__ int64_t tab_scan(int B, int32_t most, int32_t* dst, int64_t* red, F f) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int per = (B + 255) / 256, b0 = tid * per, b1 = min(b0 + per, B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += f(b);
  int64_t inc = mine;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t x = __shfl_up((long long)inc, m);
    if (lane >= m) inc += x;
  }
  __syncthreads();  // `red` of an earlier scan has been read
  if (lane == 63) red[wv] = inc;
  __syncthreads();
  int64_t at = inc - mine, all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wv) at += red[w];
    all += red[w];
  }
  for (int b = b0; b < b1; ++b) {
    dst[b] = (int32_t)min(at, (int64_t)most);
    at += f(b);
  }
  if (tid == 0) dst[B] = (int32_t)min(all, (int64_t)most);
  __syncthreads();
  return all;
}

}  // namespace htree
