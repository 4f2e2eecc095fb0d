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
// type (2^-8 of each in bf16 at most, as much as the output's own rounding; fp16
// 2^-11, or 2^-32 of the row's largest), and the sum that divides takes them rounded,
// so Values that are alike come back as they are; maxima, sums and accumulators are
// 32-bit.  Normal Values come back off by 0.0021 of the output in bf16, of which 0.0016
// is its own rounding; a second 16-bit term leaves that alone and takes 38 % longer.
//
// 8192 tokens, 32/8 heads of 128, window 4096, bf16: 398 to 428 us by card, 0.96 to
// 1.03 PFLOP/s (a large matrix product 1.34).  Power bounds it: the matrix units are
// busy half of the cycles, and the clock falls from 2.35 GHz to 1.72; waits for loads,
// barriers or LDS taken away leave the time as it is, the loads of tiles themselves
// take off an eighth.  64 rows a wave, which read LDS half as often, leave one wave a
// SIMD: a fifth longer.
#include <hip/hip_runtime.h>
#include <limits.h>

#include <type_traits>

#include "rk_paged_dev.h"

namespace {

using rk::base_of;
using rk::kFar;
using rk::kNone;
using rk::kPagedThreads;
using rk::kPagedWaves;
using rk::kSlack;
using rk::PagedArgs;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds4;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;

constexpr int kTile = 64;               // tokens
constexpr int kWaveRows = 32;
constexpr int kRows = kWaveRows * kPagedWaves;

// Instructions stay on their side.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

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

// l and two packed numbers, summed in 32 bits.
template <class DT>
__device__ __forceinline__ float add2(uint32_t w, float l) {
  if constexpr (std::is_same<DT, rk::F16>::value) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), h2{1, 1}, l, false);
  } else {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), b2{(__bf16)1.f, (__bf16)1.f}, l, false);
  }
}

// The values of this lane and of lane ^ 32, in some order.
__device__ __forceinline__ float2 both_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  const uint32_t one = r[0], two = r[1];  // (bit_cast of a vector's element takes the first)
  return make_float2(__builtin_bit_cast(float, one), __builtin_bit_cast(float, two));
}

// Where piece c of row r of a tile of Keys or Values lies in its row of CH pieces in
// LDS, and which piece lies at a place.  Rows are 16 CH bytes apart, so the rows that
// meet the same banks are every 4th, 2nd or each; they are moved apart by a rotation
// or an exclusive or, so that the 16 lanes of a read of Keys (one piece of 16 rows)
// and of Values (four rows of four pieces) have banks of their own.
template <int CH>
__device__ __forceinline__ int key_place(int c, int r) {
  if (CH == 12) return (c + (r >> 2 & 3)) % 12;
  return c ^ (CH == 16 ? r & 15 : CH == 8 ? r >> 1 & 7 : r >> 2 & 3);
}
template <int CH>
__device__ __forceinline__ int key_piece(int at, int r) {
  if (CH == 12) return (at + 12 - (r >> 2 & 3)) % 12;
  return key_place<CH>(at, r);
}
template <int CH>
__device__ __forceinline__ int value_place(int c, int r) {
  if (CH == 12) return key_place<CH>(c, r);
  return c ^ (CH == 16 ? (r & 3) << 2 : CH == 8 ? (r >> 1 & 1) << 2 : 0);
}
template <int CH>
__device__ __forceinline__ int value_piece(int at, int r) {
  return CH == 12 ? key_piece<CH>(at, r) : value_place<CH>(at, r);
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

// Whether rows of a wave (positions lo_p .. hi_p) may be NaN for what the products of
// its tiles added to what the formula says, a weight of zero times something that is not
// finite: a token without a page; one that some row does not see, with such a Value; an
// infinite Value whose weight is zero in 16 bits alone; a Key that is not finite among
// the first eight channels, which are read again past D where D is no multiple of 16.
// The tiles' last token stands behind itself too, in the rest of its tile, where nobody
// sees it.
template <class DT>
__device__ __forceinline__ bool nan_by_zero(const PagedArgs& a, int b, rk::Seen<kTile> seen, int i0, int i1, int h, int lo_p,
                                      int hi_p, int last) {
  constexpr uint32_t kExponent = std::is_same<DT, rk::F16>::value ? 0x7c00 : 0x7f80;
  auto odd_piece = [](const uint16_t* x, bool infinite) {  // of eight: not finite, or infinite
    const uint4 y = *(const uint4*)x;
    const uint32_t bits = infinite ? 0x7fff : kExponent;
    bool odd = false;
    for (const uint32_t w : {y.x, y.y, y.z, y.w}) odd |= (w & bits) == kExponent || (w >> 16 & bits) == kExponent;
    return odd;
  };
  for (int i = i0; i < i1; ++i) {
    const int j = seen.token(i) + (threadIdx.x & 63);
    bool odd = false;
    if (j <= last) {
      const uint32_t page = rk::page_of(a.map, b, j);
      const int64_t at = j & ((1u << a.map.shift) - 1);
      odd = page >= (uint32_t)a.map.pages;
      if (!odd && a.D % 16) odd = odd_piece((const uint16_t*)a.k + h * a.k_sh + (int64_t)page * a.k_sp + at * a.k_ss, false);
      const bool seen_by_all = j <= lo_p && (hi_p - j < a.window || j < a.sinks);
      const bool repeated = j == last && (last + 1) % kTile != 0;
      if (!odd) {
        const uint16_t* v = (const uint16_t*)a.v + h * a.v_sh + (int64_t)page * a.v_sp + at * a.v_ss;
        for (int c = 0; c < a.D; c += 8) odd |= odd_piece(v + c, seen_by_all && !repeated);
      }
    }
    if (__any(odd)) return true;
  }
  return false;
}

// One row by one wave, over the tokens that it sees alone (m: the score that weights
// are against): for Values that are not finite, until all its channels are NaN.  A
// lane forms the weight of one token of a tile, and sums two channels over all of them.
template <class DT>
__device__ __forceinline__ void sum_row(const PagedArgs& a, int b, Queries qs, rk::Seen<kTile> seen, int i0, int i1, int h,
                                     int row, int p0, int split, int KD, float m) {
  const int lane = threadIdx.x & 63;
  const int t = row / a.G, hq = h * a.G + row - t * a.G, p = p0 + t;
  const int c = 2 * lane;
  const bool on = c < a.D;
  const uint16_t* q = (const uint16_t*)a.q + b * a.q_sb + (qs.first + t) * a.q_st + hq * a.q_sh;
  const uint16_t* kb = (const uint16_t*)a.k + h * a.k_sh;
  const uint16_t* vb = (const uint16_t*)a.v + h * a.v_sh;
  const float q0 = on ? DT::to_f32(q[c * a.q_sd]) : 0.f, q1 = on ? DT::to_f32(q[(c + 1) * a.q_sd]) : 0.f;
  auto lane_of = [](float x, int i) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), i));
  };
  const float base = base_of(m);
  float l = 0.f, y0 = 0.f, y1 = 0.f;
  for (int i = i0; i < i1; ++i) {
    const int t0 = seen.token(i), j = t0 + lane;
    bool there = rk::sees(p, j, a.window, a.sinks);
    uint32_t page = 0;
    float w = 0.f;
    if (there) {
      page = rk::page_of(a.map, b, j);
      there = page < (uint32_t)a.map.pages;
    }
    const int64_t at = j & ((1u << a.map.shift) - 1);
    const uint16_t* k = kb + (int64_t)page * a.k_sp + at * a.k_ss;
    float s = 0.f;
    for (int d = 0; d < a.D; d += 8) {  // (by all lanes: a lane's channels of q are read by the others)
      uint4 x = make_uint4(0, 0, 0, 0);
      if (there) x = *(const uint4*)(k + d);
      const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s = __builtin_fmaf(lane_of(q0, d / 2 + e), DT::to_f32((uint16_t)u[e]), s);
        s = __builtin_fmaf(lane_of(q1, d / 2 + e), DT::to_f32((uint16_t)(u[e] >> 16)), s);
      }
    }
    if (there) w = rk::fast_exp2((s - base) * a.scale_log2 + rk::kLift<DT>);
    l += w;
    const uint64_t bits = __ballot(there);
    constexpr int kAhead = 8;
    for (int j0 = 0; j0 < kTile; j0 += kAhead) {
      uint32_t v[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        v[e] = 0;
        if (bits >> (j0 + e) & 1) {
          const uint32_t pg = (uint32_t)__builtin_amdgcn_readlane((int)page, j0 + e);
          if (on) v[e] = *(const uint32_t*)(vb + (int64_t)pg * a.v_sp + ((t0 + j0 + e) & ((1u << a.map.shift) - 1)) * a.v_ss + c);
        }
      }
#pragma unroll
      for (int e = 0; e < kAhead; ++e)
        if (bits >> (j0 + e) & 1) {
          const float x = lane_of(w, j0 + e);
          y0 = __builtin_fmaf(x, DT::to_f32((uint16_t)v[e]), y0);
          y1 = __builtin_fmaf(x, DT::to_f32((uint16_t)(v[e] >> 16)), y1);
        }
    }
    if (__all(!on || (y0 != y0 && y1 != y1))) break;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) l += rk::shfl_xor(l, d);
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

// Waves of a SIMD: what the accumulators of the channels leave room for (64
// channels, 8192 tokens: 277 us with two, 262 with three).
constexpr int waves_of(int KC) { return KC <= 4 ? 3 : 2; }

// KC: blocks of 16 channels.
template <class DT, int KC>
__global__ __launch_bounds__(kPagedThreads, waves_of(KC)) void window_kernel(const PagedArgs a) {
  constexpr int NB = (KC + 1) / 2;     // blocks of 32 channels
  constexpr int CH = 4 * NB;           // 16-byte pieces of a row in LDS
  constexpr int Pitch = CH * 16;              // bytes
  constexpr int Loads = NB;  // of a wave for a tile's Keys
  // two tiles; arrays of their own, so that reads of one do not wait for loads into the other
  __shared__ __align__(16) char s_k0[kTile * Pitch], s_k1[kTile * Pitch], s_v0[kTile * Pitch], s_v1[kTile * Pitch];
  __shared__ int s_wave[kPagedWaves], s_found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, col = lane & 31;
  const int h = blockIdx.x % a.H;
  // The last tokens see the most, so they begin first.  Where all workgroups begin at
  // once, the tiles are taken from all requests in turn, and every second workgroup of a
  // CU counts from the other end.
  int rest = blockIdx.x / a.H;
  const auto snake = [&](int n) {
    if (!a.round) return;
    const int turn = rest / a.round;
    if (turn & 1) rest = turn * a.round + min((turn + 1) * a.round, n) - 1 - rest;
  };
  int b, tile, split;
  if (a.map.starts) {
    auto count = [&](int i) { return (queries_of(a, i).n * a.G + kRows - 1) / kRows; };
    rk::Line<decltype(count)> line(a.map.B, count, s_wave, s_found);
    if (rest >= line.total * a.splits) return;
    snake(line.total * a.splits);
    split = rest % a.splits;
    const int slot = rest / a.splits;
    const bool across = a.round && a.map.B <= 64;
    const rk::Found f = across ? line.across(slot) : line.find(slot);
    b = f.b;
    if (b < 0) return;  // starts that do not ascend may count each token for every request
    tile = count(b) - 1 - (across ? f.before : slot - f.before);
  } else {
    const int tiles = (a.T * a.G + kRows - 1) / kRows;
    snake(gridDim.x / a.H);
    split = rest % a.splits;
    const int slot = rest / a.splits;
    b = a.round ? slot % a.map.B : slot / tiles;
    tile = tiles - 1 - (a.round ? slot / a.map.B : slot - b * tiles);
  }
  const Queries qs = queries_of(a, b);
  const int len = rk::len_of(a.map, b);
  const int p0 = len - qs.n;  // position of the first new token
  const int row0 = tile * kRows, rows = min(qs.n * a.G - row0, kRows);
  const int lo_p = max(p0 + row0 / a.G, 0), hi_p = p0 + (row0 + rows - 1) / a.G;
  const rk::Seen<kTile> seen(lo_p, hi_p, a.window, a.sinks);
  const int i0 = (int)((int64_t)seen.blocks * split / a.splits);
  const int i1 = a.map.pages > 0 ? (int)((int64_t)seen.blocks * (split + 1) / a.splits) : i0;

  // the wave's rows: this lane's query and its position
  const int r = wave * kWaveRows + col;
  const bool mine = r < rows;
  const int t = (row0 + r) / a.G, hq = h * a.G + (row0 + r) - t * a.G;
  const int p = mine ? p0 + t : -1;
  const int w_last = min(wave * kWaveRows + kWaveRows, rows) - 1;  // the wave's last row
  const int w_lo = max(p0 + (row0 + wave * kWaveRows) / a.G, 0);
  const int w_hi = w_last < wave * kWaveRows ? -1 : p0 + (row0 + w_last) / a.G;
  uint4 q[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) {
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
  // lane l holds the page of token l of a tile, of the last token for those behind it
  auto page_at = [&](int i) { return i < i1 ? rk::page_of(a.map, b, min(seen.token(i) + lane, hi_p)) : 0u; };
  auto there_of = [&](int i, uint32_t page) {
    return (uint64_t)__ballot(page < (uint32_t)a.map.pages && seen.token(i) + lane <= hi_p);
  };
  // A wave loads 16 rows of a tile straight to LDS, a lane 16 bytes: lane l's go
  // to the l-th place of the load's part of the tile, so it asks for the piece
  // that belongs there (past D: the first one again; queries are zero there, and
  // those channels of the output are not written).  Eight rows lie in one page: one
  // scalar address for them, and the lanes' offsets, which stay from tile to tile.
  // Behind the last token its row is loaded again (its weight is zero there), and
  // where there is no page the pool's first row.
  auto row_of = [&](int s) { return (64 * s + lane) / CH; };
  auto place_of = [&](int s) { return (64 * s + lane) % CH; };
  uint32_t k_off[Loads], v_off[Loads];  // bytes
  auto offset = [&](int i, int s, int piece, int64_t ss) {
    const int row = row_of(s), last = hi_p - seen.token(i) - 16 * wave - (row & 8);
    return 2 * ((uint32_t)min(row & 7, max(last, 0)) * (uint32_t)ss + 8 * (8 * piece < a.D ? piece : 0));
  };
  auto k_offsets = [&](int i) {
#pragma unroll
    for (int s = 0; s < Loads; ++s) k_off[s] = offset(i, s, key_piece<CH>(place_of(s), row_of(s)), a.k_ss);
  };
  auto v_offsets = [&](int i) {
#pragma unroll
    for (int s = 0; s < Loads; ++s) v_off[s] = offset(i, s, value_piece<CH>(place_of(s), row_of(s)), a.v_ss);
  };
  struct Eight {
    const char* at[2];
  };
  auto rows_at = [&](int i, uint32_t page, const uint16_t* src, int64_t sp, int64_t ss) {
    const int t0 = seen.token(i) + 16 * wave;
    Eight r;
    if (t0 + 15 <= hi_p && a.map.shift > 3) {
      const uint32_t pg = (uint32_t)__builtin_amdgcn_readlane((int)page, 16 * wave);
      const int64_t row = t0 & ((1u << a.map.shift) - 1);
      const bool ok = pg < (uint32_t)a.map.pages;
      r.at[0] = (const char*)(src + (ok ? pg : 0u) * sp + (ok ? row : 0) * ss);
      r.at[1] = r.at[0] + 16 * ss;
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t pg = (uint32_t)__builtin_amdgcn_readlane((int)page, 16 * wave + 8 * e);
        const int64_t row = min(t0 + 8 * e, hi_p) & ((1u << a.map.shift) - 1);
        const bool ok = pg < (uint32_t)a.map.pages;
        r.at[e] = (const char*)(src + (ok ? pg : 0u) * sp + (ok ? row : 0) * ss);
      }
    }
    return r;
  };
  auto load = [&](char* dst, const Eight& r, int s, uint32_t off) {
    constexpr int Half = 8 * CH;  // lanes of eight rows
    const char* from = 64 * s >= Half ? r.at[1] : r.at[0];
    if (64 * s < Half && 64 * s + 64 > Half) from = 64 * s + lane < Half ? r.at[0] : r.at[1];
    __builtin_amdgcn_global_load_lds((global_ptr)(from + off), (lds_ptr)(dst + 16 * wave * Pitch + s * 1024), 16, 0, 0);
  };
  auto load_k = [&](char* dst, const Eight& r, int s) { load(dst, r, s, k_off[s]); };
  auto load_v = [&](char* dst, const Eight& r, int s) { load(dst, r, s, v_off[s]); };
  int k_at[KC], v_at[NB][2];  // of this lane's reads of a tile; Values: eight rows on
#pragma unroll
  for (int c = 0; c < KC; ++c) k_at[c] = col * Pitch + (key_place<CH>(2 * c + hi, col) << 4);
#pragma unroll
  for (int c = 0; c < NB; ++c) {
    // lane i of 16 addresses row i / 4, four channels from 4 (i % 4), and gets channel i of four rows
    const int row = 4 * hi + ((lane & 15) >> 2), piece = 4 * c + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    v_at[c][0] = row * Pitch + (value_place<CH>(piece, row) << 4) + 8 * (lane & 1);
    v_at[c][1] = CH == 12 ? (row + 8) * Pitch + (value_place<CH>(piece, row + 8) << 4) + 8 * (lane & 1)
                          : v_at[c][0] + 8 * Pitch;
  }
  // Scores of a tile: products of two chains, reads a few products ahead.
  auto scores = [&](const char* sk, f32x16 (&n)[2]) {
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e) n[tb][e] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
        n[tb] = mfma32<DT>(*(const uint4*)(sk + k_at[c] + 32 * tb * Pitch), q[c], n[tb]);
  };
  // -inf where a row does not see the token.
  auto mask = [&](int i, uint32_t page, f32x16 (&n)[2]) {
    const int t0 = seen.token(i);
    const uint64_t there = there_of(i, page);
    if (there == ~0ull && t0 + kTile - 1 <= w_lo && (w_hi - t0 < a.window || t0 + kTile <= a.sinks)) return;
    asm volatile("");  // a branch: most tiles are whole, and the masks cost more than the scores
    const uint64_t mine_there = there >> (4 * hi);
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = 32 * tb + 8 * (e >> 2) + (e & 3);
        const bool on = rk::sees(p, t0 + 4 * hi + k, a.window, a.sinks) && (mine_there >> k & 1);
        n[tb][e] = on ? n[tb][e] : kNone;
      }
  };
  float base = 0.f;  // what the weights are against, scaled
  auto top_of = [&](const f32x16 (&n)[2]) {
    float top = kNone;
#pragma unroll
    for (int tb = 0; tb < 2; ++tb)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, n[tb][e]);
    return top;
  };
  // The next tile's scores are known: what weights are against, and the sums so far
  // against that.
  auto rebase = [&](float top, f32x16 (&n)[2]) {
    const float2 tops = both_halves(top);
    top = fmaxf(tops.x, tops.y);
    // Weights are taken against an earlier maximum while they stay below 2^8: any
    // base gives the same quotient, and few tiles raise the maximum by as much.
    if (__any((top - m) * a.scale_log2 > kSlack)) {
      asm volatile("");
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
    base = base_of(m) * a.scale_log2;
    if (__any(fabsf(base) > kFar)) {
      asm volatile("");
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int e = 0; e < 16; ++e) n[tb][e] -= base_of(m);
      base = 0.f;
    }
    base -= rk::kLift<DT>;
  };
  // Weight k of a tile's 32 in this lane, pairs of them in the products' type.
  auto weight = [&](const f32x16 (&n)[2], float (&y)[32], uint32_t (&w)[16], int k) {
    y[k] = rk::fast_exp2(__builtin_fmaf(n[k >> 4][k & 15], a.scale_log2, -base));
    if (k & 1) {
      w[k >> 1] = DT::pack2(y[k - 1], y[k]);
      asm volatile("" : "+v"(w[k >> 1]));  // here, and not where it is used
    }
  };
  auto value_at = [&](const char* sv, int g, int c) {  // 16 tokens by 32 channels
    const char* at = sv + 16 * g * Pitch;
    const uint2 u0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + v_at[c][0])));
    const uint2 u1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + v_at[c][1])));
    return make_uint4(u0.x, u0.y, u1.x, u1.y);
  };
  if (i0 < i1) {
    // pages of tiles i + 1 (Values to come), i + 2 (Keys to come) and i + 3
    const int end = i1 - 1;
    uint32_t page0 = page_at(i0), page1 = page_at(min(i0 + 1, end)), page2 = page_at(min(i0 + 2, end));
    f32x16 s[2];
    {
      k_offsets(i0);
      const Eight k0 = rows_at(i0, page0, kb, a.k_sp, a.k_ss), v0 = rows_at(i0, page0, vb, a.v_sp, a.v_ss);
#pragma unroll
      for (int r = 0; r < Loads; ++r) load_k(s_k0, k0, r);
      v_offsets(i0);
#pragma unroll
      for (int r = 0; r < Loads; ++r) load_v(s_v0, v0, r);
      loads_done();
      __syncthreads();
      k_offsets(min(i0 + 1, end));
      const Eight k1 = rows_at(min(i0 + 1, end), page1, kb, a.k_sp, a.k_ss);
#pragma unroll
      for (int r = 0; r < Loads; ++r) load_k(s_k1, k1, r);
      scores(s_k0, s);
      mask(i0, page0, s);
      rebase(top_of(s), s);
    }
    // Tile i's weights and products with Values, beside the products of tile i + 1's
    // scores and the loads of what the next step takes.
    auto step = [&](int i, const char* next_k, const char* sv, char* k_to, char* v_to, auto last) {
      constexpr bool kLast = decltype(last)::value;
      loads_done();
      __syncthreads();  // these tiles are there for all waves, and the last ones have been read by all
      const int ik = min(i + 2, end);
      uint32_t page3 = 0;
      Eight rk_, rv;
      if (!kLast) {
        page3 = page_at(min(i + 3, end));
        if (ik == end) {
          asm volatile("");  // a branch
          k_offsets(ik);
          if (i + 1 == end) v_offsets(end);
        }
        rk_ = rows_at(ik, page2, kb, a.k_sp, a.k_ss);
        rv = rows_at(i + 1, page1, vb, a.v_sp, a.v_ss);
      }
      f32x16 n[2];
      float y[32];
      uint32_t w[16];
      // Two products at a time, and what the other units do meanwhile: a product
      // takes the matrix unit 32 cycles, an exponential its own 16.  The fences keep
      // the mixture as it is written.
      if (!kLast) {
        uint4 k0[KC], k1[KC];
        auto read = [&](int c) {
          k0[c] = *(const uint4*)(next_k + k_at[c]);
          k1[c] = *(const uint4*)(next_k + k_at[c] + 32 * Pitch);
        };
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int e = 0; e < 16; ++e) n[tb][e] = 0.f;
        read(0);
        if (KC > 1) read(1);
        fence();
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          if (c + 2 < KC) read(c + 2);
          n[0] = mfma32<DT>(k0[c], q[c], n[0]);
          n[1] = mfma32<DT>(k1[c], q[c], n[1]);
#pragma unroll
          for (int r = 0; r < 2 * Loads; ++r)
            if (r * KC / (2 * Loads) == c) r & 1 ? load_k(k_to, rk_, r >> 1) : load_v(v_to, rv, r >> 1);
#pragma unroll
          for (int k = 0; k < 24; ++k)
            if (k * KC / 24 == c) weight(s, y, w, k);
          fence();
        }
        mask(i + 1, page1, n);
      } else {
#pragma unroll
        for (int k = 0; k < 24; ++k) weight(s, y, w, k);
      }
      float top = kNone;
      {
        constexpr int kProducts = 4 * NB;  // (g, c): g 16 tokens, c 32 channels
        uint4 v[kProducts];
        auto read = [&](int j) { v[j] = value_at(sv, j / NB, j % NB); };
#pragma unroll
        for (int j = 0; j < 4; ++j) read(j);
        fence();
#pragma unroll
        for (int j = 0; j < kProducts; j += 2) {
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            if (j + d + 4 < kProducts) read(j + d + 4);
            const int g = (j + d) / NB, c = (j + d) % NB;
            o[c] = mfma32<DT>(v[j + d], make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]), o[c]);
          }
#pragma unroll
          for (int k = 24; k < 32; ++k)
            if ((k - 24) * (3 * NB / 2) / 8 == j / 2) weight(s, y, w, k);
          // (here the sums take no time; beside the scores' products 3 % of it)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (k * (kProducts / 2) / 16 == j / 2) l = add2<DT>(w[k], l);
          if (!kLast) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k * (kProducts / 2) / 32 == j / 2) top = fmaxf(top, n[k >> 4][k & 15]);
          }
          fence();
        }
      }
      if (!kLast) {
        rebase(top, n);
        s[0] = n[0];
        s[1] = n[1];
      }
      page1 = page2;
      page2 = page3;
    };
    int i = i0;
    for (; i + 2 < i1; i += 2) {
      step(i, s_k1, s_v0, s_k0, s_v1, std::false_type{});
      step(i + 1, s_k0, s_v1, s_k1, s_v0, std::false_type{});
    }
    if (i + 1 < i1) {
      step(i, s_k1, s_v0, s_k0, s_v1, std::false_type{});
      step(i + 1, s_k0, s_v1, s_k1, s_v0, std::true_type{});
    } else {
      step(i, s_k1, s_v0, s_k0, s_v1, std::true_type{});
    }
  }
  const float2 sums = both_halves(l);
  l = sums.x + sums.y;
  // Weight 0 times an infinity or a NaN is a NaN: a tile's Values reach rows that do
  // not see them, or by a weight that is too small for 16 bits.  Where there are such,
  // rows that are NaN are summed again from what they see.
  bool nan = l != l;
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) nan |= o[c][e] != o[c][e];
  const uint64_t odd = __ballot(mine && nan);
  uint32_t again = (uint32_t)odd | (uint32_t)(odd >> 32);
  if (again && !nan_by_zero<DT>(a, b, seen, i0, i1, h, p0 + (row0 + wave * kWaveRows) / a.G, w_hi, hi_p)) again = 0;
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
  constexpr int kAhead = 4;
  float m = kNone, l = 0.f, y0 = 0.f, y1 = 0.f;
  for (int s0 = 0; s0 < a.splits; s0 += kAhead) {
    float2 ml[kAhead], x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t rec = min(s0 + k, a.splits - 1) * rows + row;
      ml[k] = *(const float2*)(a.ml + 2 * rec);
      x[k] = c < a.D ? *(const float2*)(a.acc + rec * KD + c) : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (s0 + k >= a.splits) break;
      const float top = fmaxf(m, ml[k].x), base = base_of(top);
      const float f0 = rk::fast_exp2(m - base), f1 = rk::fast_exp2(ml[k].x - base);
      l = l * f0 + ml[k].y * f1;
      y0 = y0 * f0 + x[k].x * f1;
      y1 = y1 * f0 + x[k].y * f1;
      m = top;
    }
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

int window_per_cu(const PagedArgs& a) { return waves_of((a.D + 15) / 16); }

int window_launch(const PagedArgs& a, int32_t dtype, hipStream_t s) {
  const int64_t grid = window_slots(a) * a.H * a.splits, rows = a.N * a.Hq;
  auto on = [&](auto dt, auto kc) {
    constexpr int KC = decltype(kc)::value;
    hipLaunchKernelGGL((window_kernel<decltype(dt), KC>), dim3((unsigned)grid), dim3(kPagedThreads), 0, s, a);
    if (a.splits > 1)
      hipLaunchKernelGGL((window_join_kernel<decltype(dt)>), dim3((unsigned)((rows + kPagedWaves - 1) / kPagedWaves)),
                         dim3(kPagedThreads), 0, s, a, 32 * ((KC + 1) / 2));
  };
  auto by_dim = [&](auto dt) {
    switch ((a.D + 15) / 16) {
      case 1: return on(dt, std::integral_constant<int, 1>{});
      case 2: return on(dt, std::integral_constant<int, 2>{});
      case 3: return on(dt, std::integral_constant<int, 3>{});
      case 4: return on(dt, std::integral_constant<int, 4>{});
      case 5: return on(dt, std::integral_constant<int, 5>{});
      case 6: return on(dt, std::integral_constant<int, 6>{});
      case 7: return on(dt, std::integral_constant<int, 7>{});
      default: return on(dt, std::integral_constant<int, 8>{});
    }
  };
  dtype == RK_F16 ? by_dim(F16{}) : by_dim(BF16{});
  return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_HIP;
}

}  // namespace rk
