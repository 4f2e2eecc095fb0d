// rk_paged_dev.h -- device code that the kernels of rk_paged.hip and
// rk_window.hip share: what a token sees, and how the work of requests of
// different lengths is divided.
#pragma once

#include <type_traits>

#include "rk_common.h"
#include "rk_paged.h"

namespace rk {

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = 4;
constexpr float kNone = -__builtin_inff();
constexpr float kSlack = 8.f;    // log2 of what weights may grow to
constexpr float kFar = 16384.f;  // a base of scores, in log2, that is rounded by 2^-11 at most

// log2 of what all weights are raised by, which the quotient does not show.  fp16 ends
// at 2^-24, so a weight loses up to 2^-25 whatever its size; weights are 2^kSlack at
// most, so another 2^7 fit below 65504, and the loss is 2^-32 of the largest weight.
template <class DT>
constexpr float kLift = std::is_same<DT, F16>::value ? 7.f : 0.f;

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

// Sum over the wave's lanes up to this one.
__device__ __forceinline__ int wave_sum_to(int n) {
  n += __builtin_amdgcn_update_dpp(0, n, 0x111, 0xf, 0xf, true);  // one lane of the row before, then two, ..
  n += __builtin_amdgcn_update_dpp(0, n, 0x112, 0xf, 0xf, true);
  n += __builtin_amdgcn_update_dpp(0, n, 0x114, 0xf, 0xf, true);
  n += __builtin_amdgcn_update_dpp(0, n, 0x118, 0xf, 0xf, true);
  n += __builtin_amdgcn_update_dpp(0, n, 0x142, 0xa, 0xf, false);  // the last lane of the row before, to rows 1 and 3
  n += __builtin_amdgcn_update_dpp(0, n, 0x143, 0xc, 0xf, false);  // of the first half, to the second
  return n;
}

struct Found {
  int b, before;  // a request (below zero: none), and the pieces before it
};

// Work of requests 0 .. B - 1, count(b) pieces each, laid end to end: the sum, and
// the request that a piece belongs to.  Up to 64 requests every wave looks for
// itself, without a barrier.
template <class F>
struct Line {
  F count;
  int B, total;
  int mine, to;  // up to 64 requests: the lane's pieces, and those up to them
  int *s_wave, *s_found;

  __device__ __forceinline__ Line(int B, F count, int* s_wave, int* s_found)
      : count(count), B(B), s_wave(s_wave), s_found(s_found) {
    if (B <= 64) {
      const int lane = threadIdx.x & 63;
      mine = lane < B ? count(lane) : 0;
      to = wave_sum_to(mine);
      total = __builtin_amdgcn_readlane(to, 63);
    } else {
      int sum = 0;
      for (int b = threadIdx.x; b < B; b += kPagedThreads) sum += count(b);
      scan_before(sum, s_wave, &total);
    }
  }

  // Up to 64 requests, the first piece of each before the second ones: the request of
  // piece `at`, and how many of its own come before it.
  __device__ __forceinline__ Found across(int at) const {
    auto within = [&](int n) { return __builtin_amdgcn_readlane(wave_sum_to(min(mine, n)), 63); };  // the first n of each
    int low = 0, high = 1;
    while (within(high) <= at) {
      low = high;
      high *= 2;
    }
    while (high - low > 1) {
      const int mid = (low + high) / 2;
      if (within(mid) <= at) low = mid; else high = mid;
    }
    const int left = at - within(low);  // (by all lanes, ahead of any condition)
    const uint64_t more = __ballot(mine > low);
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(more >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)more, 0));
    return {__builtin_ctzll(__ballot((mine > low) & (rank == left))), low};
  }

  // `at` below the sum; none where counts of more than 64 requests add up to 2^31 or more.
  __device__ __forceinline__ Found find(int at) {
    if (B <= 64) {
      const int b = __builtin_ctzll(__ballot(at < to));
      return {b, __builtin_amdgcn_readlane(to - mine, b)};
    }
    if (threadIdx.x == 0) s_found[0] = -1;  // (the scan's barriers stand between this and the next)
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += kPagedThreads) {
      const int b = b0 + threadIdx.x;
      const int n = b < B ? count(b) : 0;
      int sum;
      const int first = before + scan_before(n, s_wave, &sum);
      if (at >= first && at < first + n) {
        s_found[0] = b;
        s_found[1] = first;
      }
      before += sum;
      if (at < before) break;
    }
    __syncthreads();
    return {s_found[0], s_found[1]};
  }
};

}  // namespace rk
