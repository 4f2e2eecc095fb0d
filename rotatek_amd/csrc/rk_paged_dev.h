// rk_paged_dev.h -- device code that the kernels of rk_paged.hip and
// rk_window.hip share: what a token sees, and how the work of requests of
// different lengths is divided.
#pragma once

#include "rk_common.h"
#include "rk_paged.h"

namespace rk {

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = 4;
constexpr float kNone = -__builtin_inff();
constexpr float kSlack = 8.f;    // log2 of what weights may grow to
constexpr float kFar = 16384.f;  // a base of scores, in log2, that is rounded by 2^-11 at most

// 2^(x - m), and the maximum to subtract where nothing counted yet: -inf - -inf
// would be NaN.
__device__ __forceinline__ float base_of(float m) { return m == kNone ? 0.f : m; }

// Sum over the workgroup's threads before this one, and the whole sum.
__device__ __forceinline__ int scan_before(int n, int* s_wave, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int at = n;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int up = __shfl_up(at, d, 64);
    if (lane >= d) at += up;
  }
  __syncthreads();  // the last call's sums have been read
  if (lane == 63) s_wave[wave] = at;
  __syncthreads();
  int before = at - n, sum = 0;
#pragma unroll
  for (int w = 0; w < kPagedWaves; ++w) {
    if (w < wave) before += s_wave[w];
    sum += s_wave[w];
  }
  *total = sum;
  return before;
}

// Work of requests 0 .. B - 1, count(b) pieces each, laid end to end: their
// sum.
template <class F>
__device__ __forceinline__ int pieces_of_all(int B, F count, int* s_wave) {
  int sum = 0;
  for (int b = threadIdx.x; b < B; b += kPagedThreads) sum += count(b);
  int total;
  scan_before(sum, s_wave, &total);
  return total;
}

struct Found {
  int b, before;  // the request, and the pieces before it
};

// The request that piece `at` (below the sum) belongs to.
template <class F>
__device__ __forceinline__ Found request_at(int B, F count, int at, int* s_wave, int* s_found) {
  int before = 0;
  for (int b0 = 0; b0 < B; b0 += kPagedThreads) {
    const int b = b0 + threadIdx.x;
    const int n = b < B ? count(b) : 0;
    int total;
    const int mine = before + scan_before(n, s_wave, &total);
    if (at >= mine && at < mine + n) {
      s_found[0] = b;
      s_found[1] = mine;
    }
    before += total;
    if (at < before) break;
  }
  __syncthreads();
  return {s_found[0], s_found[1]};
}

}  // namespace rk
