// rk_window.hip -- attention of many new tokens, each over the last `window`
// tokens before it and the first `sinks` of its request, on MI355X (gfx950):
// the kernels of rk_paged_attention with starts and of rk_window_attention.
//
// A workgroup takes 128 rows of one KV head; a row is a (new token, query head
// of the group) pair, so a group's heads share every Key and Value tile and a
// tile's rows are as few tokens apart as can be.  Tiles of 64 tokens go through
// LDS, two at a time: the next one's loads are in flight while this one is
// multiplied.  A wave keeps 32 rows: S^T = K Q^T (32 tokens by 32 rows a
// product) leaves each lane the scores of one row, eight of 16 tokens in the
// order in which O^T = V^T P^T takes them, so that weights stay where they are;
// V^T is read by the transposing LDS load.  Weights are rounded to the inputs'
// type (2^-9 of each in bf16, as much as the output's own rounding); maxima,
// sums and accumulators are 32-bit.
#include <hip/hip_runtime.h>
#include <limits.h>

#include <type_traits>

#include "rk_paged_dev.h"

namespace {

using rk::base_of;
using rk::kNone;
using rk::kPagedThreads;
using rk::kPagedWaves;
using rk::PagedArgs;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds4;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;

constexpr int kTile = 64;               // tokens
constexpr int kWaveRows = 32;
constexpr int kRows = kWaveRows * kPagedWaves;
constexpr float kSlack = 8.f;           // log2 of what weights may grow to
constexpr float kFar = 16384.f;         // a base that is rounded by 2^-11 at most

// The wave's loads to LDS have arrived.
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <class DT>
__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
  if constexpr (std::is_same<DT, rk::F16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(rk::f16x8, a), __builtin_bit_cast(rk::f16x8, b),
                                                  c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(rk::bf16x8, a),
                                                   __builtin_bit_cast(rk::bf16x8, b), c, 0, 0, 0);
}

// Where the pieces of a row of Keys or Values lie in LDS: piece c at c ^ swap.
template <int CH>
__device__ __forceinline__ int key_swap(int row) {
  return CH == 16 ? row & 15 : (row >> 1) & 7;
}
template <int CH>
__device__ __forceinline__ int value_swap(int row) {
  return CH == 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
}

// New tokens of request b: first and how many.
struct Queries {
  int64_t first;
  int n;
};
__device__ __forceinline__ Queries queries_of(const PagedArgs& a, int b) {
  if (!a.map.starts) return {0, a.T};
  const int64_t s = max(a.map.starts[b], 0), e = min((int64_t)a.map.starts[b + 1], a.N);
  return {s, (int)max(e - s, (int64_t)0)};
}

// One row by one wave, two channels a lane, over the tokens that it sees alone
// (m: the score that weights are against): any cost, for Values that are not
// finite.
template <class DT>
__device__ __forceinline__ void sum_row(const PagedArgs& a, int b, Queries qs, rk::Seen<kTile> seen, int i0, int i1, int h,
                                     int row, int p0, int split, int KD, float m) {
  const int t = row / a.G, hq = h * a.G + row - t * a.G, p = p0 + t;
  const int c = 2 * (threadIdx.x & 63);
  const bool on = c < a.D;
  const uint16_t* q = (const uint16_t*)a.q + b * a.q_sb + (qs.first + t) * a.q_st + hq * a.q_sh;
  const uint16_t* kb = (const uint16_t*)a.k + h * a.k_sh;
  const uint16_t* vb = (const uint16_t*)a.v + h * a.v_sh;
  const float q0 = on ? DT::to_f32(q[c * a.q_sd]) : 0.f, q1 = on ? DT::to_f32(q[(c + 1) * a.q_sd]) : 0.f;
  const float base = base_of(m);
  float l = 0.f, y0 = 0.f, y1 = 0.f;
  for (int i = i0; i < i1; ++i) {
    const int t0 = seen.token(i);
    for (int j = t0; j < t0 + kTile; ++j) {
      if (!rk::sees(p, j, a.window, a.sinks)) continue;
      const uint32_t page = rk::page_of(a.map, b, j);
      if (page >= (uint32_t)a.map.pages) continue;
      const int64_t at = j & ((1u << a.map.shift) - 1);
      const uint16_t* k = kb + (int64_t)page * a.k_sp + at * a.k_ss;
      const uint16_t* v = vb + (int64_t)page * a.v_sp + at * a.v_ss;
      float s = on ? q0 * DT::to_f32(k[c]) + q1 * DT::to_f32(k[c + 1]) : 0.f;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) s += rk::shfl_xor(s, d);
      const float w = rk::fast_exp2((s - base) * a.scale_log2);
      l += w;
      if (on) {
        y0 += w * DT::to_f32(v[c]);
        y1 += w * DT::to_f32(v[c + 1]);
      }
    }
  }
  if (!on) return;
  if (a.splits > 1) {
    const int64_t rec = (int64_t)split * a.N * a.Hq + (b * (int64_t)a.T + qs.first + t) * a.Hq + hq;
    *(float2*)(a.acc + rec * KD + c) = make_float2(y0, y1);
    if (c == 0) *(float2*)(a.ml + 2 * rec) = make_float2(m * a.scale_log2, l);
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint16_t* dst = (uint16_t*)a.out + b * a.o_sb + (qs.first + t) * a.o_st + hq * a.o_sh;
  dst[c * a.o_sd] = DT::from_f32(y0 * inv);
  dst[(c + 1) * a.o_sd] = DT::from_f32(y1 * inv);
}

template <class DT, int NB>
__global__ __launch_bounds__(kPagedThreads, 2) void window_kernel(const PagedArgs a) {
  constexpr int CH = NB <= 2 ? 8 : 16;        // 16-byte pieces of a row in LDS
  constexpr int Pitch = CH * 16;              // bytes
  constexpr int Passes = kTile * CH / kPagedThreads;  // loads of a wave for a tile's Keys
  // two tiles; arrays of their own, so that reads of one do not wait for loads into the other
  __shared__ __align__(16) char s_k0[kTile * Pitch], s_k1[kTile * Pitch], s_v0[kTile * Pitch], s_v1[kTile * Pitch];
  __shared__ int s_wave[kPagedWaves], s_found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, col = lane & 31;
  const int h = blockIdx.x % a.H;
  const int rest = blockIdx.x / a.H;
  const int split = rest % a.splits, slot = rest / a.splits;
  int b, tile;
  if (a.map.starts) {
    auto count = [&](int i) { return (queries_of(a, i).n * a.G + kRows - 1) / kRows; };
    const int tiles = rk::pieces_of_all(a.map.B, count, s_wave);
    if (slot >= tiles) return;
    const rk::Found f = rk::request_at(a.map.B, count, slot, s_wave, s_found);
    b = f.b;
    tile = count(b) - 1 - (slot - f.before);
  } else {
    const int tiles = (a.T * a.G + kRows - 1) / kRows;
    b = slot / tiles;
    tile = tiles - 1 - (slot - b * tiles);  // the last tokens see the most: they begin first
  }
  const Queries qs = queries_of(a, b);
  const int len = rk::len_of(a.map, b);
  const int p0 = len - qs.n;  // position of the first new token
  const int row0 = tile * kRows, rows = min(qs.n * a.G - row0, kRows);
  const int lo_p = max(p0 + row0 / a.G, 0), hi_p = p0 + (row0 + rows - 1) / a.G;
  const rk::Seen<kTile> seen(lo_p, hi_p, a.window, a.sinks);
  const int i0 = (int)((int64_t)seen.blocks * split / a.splits);
  const int i1 = (int)((int64_t)seen.blocks * (split + 1) / a.splits);

  // the wave's rows: this lane's query and its position
  const int r = wave * kWaveRows + col;
  const bool mine = r < rows;
  const int t = (row0 + r) / a.G, hq = h * a.G + (row0 + r) - t * a.G;
  const int p = mine ? p0 + t : -1;
  const int w_last = min(wave * kWaveRows + kWaveRows, rows) - 1;  // the wave's last row
  const int w_lo = max(p0 + (row0 + wave * kWaveRows) / a.G, 0);
  const int w_hi = w_last < wave * kWaveRows ? -1 : p0 + (row0 + w_last) / a.G;
  uint4 q[2 * NB];
#pragma unroll
  for (int c = 0; c < 2 * NB; ++c) {
    const int ch = 16 * c + 8 * hi;
    q[c] = make_uint4(0, 0, 0, 0);
    if (mine && ch < a.D) {
      const uint16_t* src = (const uint16_t*)a.q + b * a.q_sb + (qs.first + t) * a.q_st + hq * a.q_sh + ch * a.q_sd;
      q[c] = a.q_vec ? rk::load8<true>(src, 1, 8) : rk::load8<false>(src, a.q_sd, 8);
    }
  }
  float m = kNone, l = 0.f;
  f32x16 o[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[c][e] = 0.f;

  const uint16_t* kb = (const uint16_t*)a.k + h * a.k_sh;
  const uint16_t* vb = (const uint16_t*)a.v + h * a.v_sh;
  // lane l holds the page of token l of a tile; one past the pool where no row sees it
  auto page_at = [&](int i) {
    const int j = seen.token(i) + lane;
    return i < i1 && j <= hi_p ? rk::page_of(a.map, b, j) : 0xffffffffu;
  };
  // A wave loads 16 rows of a tile straight to LDS, a lane 16 bytes: lane l's go
  // to the l-th place of the load's part of the tile, so it asks for the piece
  // that belongs there.  Pieces are swapped about in each row, so that the 16
  // lanes of a read of Keys (one piece of 16 rows) and of Values (four rows of
  // four pieces) meet different banks.  The rows lie in one page, or in two of
  // eight rows.
  constexpr int PerLoad = 64 / CH;  // rows
  const int lrow = lane / CH, lpc = lane % CH;
  uint32_t k_off[Passes];  // bytes
#pragma unroll
  for (int s = 0; s < Passes; ++s)
    k_off[s] = 2 * (lrow * (uint32_t)a.k_ss + 8 * (lpc ^ key_swap<CH>(PerLoad * s + lrow)));
  const uint32_t v_off = 2 * (lrow * (uint32_t)a.v_ss + 8 * (lpc ^ value_swap<CH>(lrow)));
  const bool full = a.D == 8 * CH;
  auto stage = [&](char* sk, char* sv, int i, uint32_t page, uint64_t there) {
    const int first = 16 * wave, t0 = seen.token(i) + first;
    const bool all = full && ((there >> first) & 0xffff) == 0xffff;
    const char *kp[Passes], *vp[Passes];
#pragma unroll
    for (int s = 0; s < Passes; ++s) {
      const uint32_t pg = (uint32_t)__builtin_amdgcn_readlane((int)page, first + (PerLoad * s & 8));
      const int64_t at = (t0 + PerLoad * s) & ((1u << a.map.shift) - 1);
      kp[s] = (const char*)(kb + pg * a.k_sp + at * a.k_ss);
      vp[s] = (const char*)(vb + pg * a.v_sp + at * a.v_ss);
    }
    sk += first * Pitch;
    sv += first * Pitch;
    if (all) {
#pragma unroll
      for (int s = 0; s < Passes; ++s) {
        __builtin_amdgcn_global_load_lds((global_ptr)(kp[s] + k_off[s]), (lds_ptr)(sk + s * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((global_ptr)(vp[s] + v_off), (lds_ptr)(sv + s * 1024), 16, 0, 0);
      }
      return;
    }
#pragma unroll
    for (int s = 0; s < Passes; ++s) {
      const int row = PerLoad * s + lrow;
      if (there >> (first + row) & 1) {
        if (8 * (lpc ^ key_swap<CH>(row)) < a.D)
          __builtin_amdgcn_global_load_lds((global_ptr)(kp[s] + k_off[s]), (lds_ptr)(sk + s * 1024), 16, 0, 0);
        if (8 * (lpc ^ value_swap<CH>(row)) < a.D)
          __builtin_amdgcn_global_load_lds((global_ptr)(vp[s] + v_off), (lds_ptr)(sv + s * 1024), 16, 0, 0);
      } else {
        *(uint4*)(sk + s * 1024 + 16 * lane) = make_uint4(0, 0, 0, 0);
        *(uint4*)(sv + s * 1024 + 16 * lane) = make_uint4(0, 0, 0, 0);
      }
    }
  };
  int k_at[2 * NB], v_at[NB];  // of this lane's reads of a tile
#pragma unroll
  for (int c = 0; c < 2 * NB; ++c) k_at[c] = col * Pitch + (((2 * c + hi) ^ key_swap<CH>(col)) << 4);
#pragma unroll
  for (int c = 0; c < NB; ++c) {
    // lane i of 16 addresses row i / 4, four channels from 4 (i % 4), and gets channel i of four rows
    const int row = (lane & 15) >> 2, piece = 4 * c + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    v_at[c] = (4 * hi + row) * Pitch + ((piece ^ value_swap<CH>(row)) << 4) + 8 * (lane & 1);
  }
  auto multiply = [&](const char* sk, const char* sv, int i, uint64_t there) {
    const int t0 = seen.token(i);
    // tiles that no row of the wave sees
    if (t0 > w_hi || (t0 + kTile - 1 <= w_lo - a.window && t0 >= a.sinks)) return;
    float x[2][16];
#pragma unroll
    for (int tb = 0; tb < 2; ++tb) {
      f32x16 sc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
      for (int c = 0; c < 2 * NB; ++c) {
        const uint4 kf = *(const uint4*)(sk + k_at[c] + 32 * tb * Pitch);
        sc = mfma32<DT>(kf, q[c], sc);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) x[tb][e] = sc[e];
    }
    const bool whole = there == ~0ull && t0 + kTile - 1 <= w_lo && (w_hi - t0 < a.window || t0 + kTile <= a.sinks);
    if (!whole) {
      asm volatile("");  // a branch: most tiles are whole, and the masks cost more than the scores
      const uint64_t mine_there = there >> (4 * hi);
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = 32 * tb + 8 * (e >> 2) + (e & 3);
          const bool on = rk::sees(p, t0 + 4 * hi + k, a.window, a.sinks) && (mine_there >> k & 1);
          x[tb][e] = on ? x[tb][e] : kNone;
        }
    }
    float top = kNone;
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, x[tb][e]);
    top = fmaxf(top, rk::shfl_xor(top, 32));
    // Weights are taken against an earlier maximum while they stay below 2^8: any
    // base gives the same quotient, and few tiles raise the maximum by as much.
    if (__any((top - m) * a.scale_log2 > kSlack)) {
      const float m_new = fmaxf(m, top), keep = rk::fast_exp2((m - base_of(m_new)) * a.scale_log2);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[c][e] *= keep;
    }
    // Scale and base in one product, whose base is rounded: all of a row's weights
    // take the same factor 2^(2^-24 base) from it, which far scores would make large.
    float base = base_of(m) * a.scale_log2;
    if (__any(fabsf(base) > kFar)) {
      asm volatile("");
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[tb][e] -= base_of(m);
      base = 0.f;
    }
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[tb][e] = rk::fast_exp2(__builtin_fmaf(x[tb][e], a.scale_log2, -base));
        l += x[tb][e];
      }
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float* y = x[tb] + 8 * u;
        const uint4 w = make_uint4(DT::pack2(y[0], y[1]), DT::pack2(y[2], y[3]), DT::pack2(y[4], y[5]),
                                   DT::pack2(y[6], y[7]));
#pragma unroll
        for (int c = 0; c < NB; ++c) {
          const char* at = sv + v_at[c] + (32 * tb + 16 * u) * Pitch;
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * Pitch));
          const uint2 u0 = __builtin_bit_cast(uint2, v0), u1 = __builtin_bit_cast(uint2, v1);
          o[c] = mfma32<DT>(make_uint4(u0.x, u0.y, u1.x, u1.y), w, o[c]);
        }
      }
  };
  if (i0 < i1) {
    // pieces past D are never loaded: they stay zero
    if (a.D < 8 * CH) {
      for (int at = 16 * tid; at < kTile * Pitch; at += 16 * kPagedThreads) {
        *(uint4*)(s_k0 + at) = *(uint4*)(s_k1 + at) = *(uint4*)(s_v0 + at) = *(uint4*)(s_v1 + at) =
            make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
    }
    auto is_there = [&](uint32_t page) { return (uint64_t)__ballot(page < (uint32_t)a.map.pages); };
    uint32_t page = page_at(i0), page_next = page_at(i0 + 1);
    uint64_t there = is_there(page);
    stage(s_k0, s_v0, i0, page, there);
    auto step = [&](int i, const char* sk, const char* sv, char* next_k, char* next_v) {
      loads_done();
      __syncthreads();  // this tile is there for all waves, and the last one has been read by all
      const uint64_t here = there;
      page = page_next;
      there = is_there(page);
      page_next = page_at(i + 2);
      if (i + 1 < i1) stage(next_k, next_v, i + 1, page, there);
      multiply(sk, sv, i, here);
    };
    for (int i = i0; i < i1; i += 2) {
      step(i, s_k0, s_v0, s_k1, s_v1);
      if (i + 1 < i1) step(i + 1, s_k1, s_v1, s_k0, s_v0);
    }
  }
  l += rk::shfl_xor(l, 32);
  // Weight 0 times an infinity or a NaN is a NaN: a tile's Values reach rows
  // that do not see them.  Rows that are not finite are summed again from what
  // they see.
  float probe = l * 0.f;
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) probe += o[c][e] * 0.f;
  const uint64_t odd = __ballot(mine && probe != 0.f);
  uint32_t again = (uint32_t)odd | (uint32_t)(odd >> 32);
  const bool done = again >> col & 1;
  while (again) {
    const int rr = __builtin_ctz(again);
    again &= again - 1;
    sum_row<DT>(a, b, qs, seen, i0, i1, h, row0 + wave * kWaveRows + rr, p0, split, 32 * NB,
                __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, m), rr)));
  }
  if (!mine || done) return;
  if (a.splits > 1) {
    const int64_t rec = (int64_t)split * a.N * a.Hq + (b * (int64_t)a.T + qs.first + t) * a.Hq + hq;
    float* dst = a.acc + rec * (32 * NB);
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(float4*)(dst + 32 * c + 2 * e + 4 * hi) = make_float4(o[c][e], o[c][e + 1], o[c][e + 2], o[c][e + 3]);
    if (hi == 0) *(float2*)(a.ml + 2 * rec) = make_float2(m * a.scale_log2, l);
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint16_t* dst = (uint16_t*)a.out + b * a.o_sb + (qs.first + t) * a.o_st + hq * a.o_sh;
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int ch = 32 * c + 2 * e + 4 * hi;
      if (ch >= a.D) continue;
      const float y[4] = {o[c][e] * inv, o[c][e + 1] * inv, o[c][e + 2] * inv, o[c][e + 3] * inv};
      if (a.o_vec) {
        *(uint2*)(dst + ch) = make_uint2(DT::pack2(y[0], y[1]), DT::pack2(y[2], y[3]));
      } else {
#pragma unroll
        for (int f = 0; f < 4; ++f) dst[(ch + f) * a.o_sd] = DT::from_f32(y[f]);
      }
    }
}

// Joins the splits of a row: a wave each.
template <class DT>
__global__ __launch_bounds__(kPagedThreads) void window_join_kernel(const PagedArgs a, int KD) {
  const int64_t rows = a.N * a.Hq;
  const int64_t row = (int64_t)blockIdx.x * kPagedWaves + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t n = row / a.Hq, hq = row - n * a.Hq;
  int64_t b = 0, t = n;
  if (a.map.starts) {
    b = rk::request_of(a.map.starts, a.map.B, n);
    if (n < a.map.starts[b] || n >= a.map.starts[b + 1]) return;  // no request's: stays as it is
    b = 0;
  } else {
    b = n / a.T;
    t = n - b * a.T;
  }
  const int c = 2 * (threadIdx.x & 63);
  float m = kNone, l = 0.f, y0 = 0.f, y1 = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const int64_t rec = s * rows + row;
    const float2 ml = *(const float2*)(a.ml + 2 * rec);
    const float2 x = c < a.D ? *(const float2*)(a.acc + rec * KD + c) : make_float2(0.f, 0.f);
    const float top = fmaxf(m, ml.x), base = base_of(top);
    const float f0 = rk::fast_exp2(m - base), f1 = rk::fast_exp2(ml.x - base);
    l = l * f0 + ml.y * f1;
    y0 = y0 * f0 + x.x * f1;
    y1 = y1 * f0 + x.y * f1;
    m = top;
  }
  if (c >= a.D) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  uint16_t* dst = (uint16_t*)a.out + b * a.o_sb + t * a.o_st + hq * a.o_sh;
  dst[c * a.o_sd] = DT::from_f32(y0 * inv);
  dst[(c + 1) * a.o_sd] = DT::from_f32(y1 * inv);
}

}  // namespace

namespace rk {

int64_t window_slots(const PagedArgs& a) {
  if (a.map.starts) return (a.N * a.G + kRows - 1) / kRows + a.map.B;
  return a.map.B * (((int64_t)a.T * a.G + kRows - 1) / kRows);
}

int window_launch(const PagedArgs& a, int32_t dtype, hipStream_t s) {
  const int64_t grid = window_slots(a) * a.H * a.splits, rows = a.N * a.Hq;
  const int NB = (a.D + 31) / 32;
  auto on = [&](auto dt, auto nb) {
    hipLaunchKernelGGL((window_kernel<decltype(dt), decltype(nb)::value>), dim3((unsigned)grid), dim3(kPagedThreads),
                       0, s, a);
    if (a.splits > 1)
      hipLaunchKernelGGL((window_join_kernel<decltype(dt)>), dim3((unsigned)((rows + kPagedWaves - 1) / kPagedWaves)),
                         dim3(kPagedThreads), 0, s, a, 32 * NB);
  };
  auto by_dim = [&](auto dt) {
    switch (NB) {
      case 1: on(dt, std::integral_constant<int, 1>{}); break;
      case 2: on(dt, std::integral_constant<int, 2>{}); break;
      case 3: on(dt, std::integral_constant<int, 3>{}); break;
      default: on(dt, std::integral_constant<int, 4>{});
    }
  };
  dtype == RK_F16 ? by_dim(F16{}) : by_dim(BF16{});
  return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_HIP;
}

}  // namespace rk
