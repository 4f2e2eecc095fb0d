// rk_paged.hip -- attention of new tokens over a paged KV cache or plain rows
// on MI355X (gfx950): the host code of rk_paged_attention and
// rk_window_attention, and the kernels of one new token a request.
//
// One token.  A request's Keys and Values are read once and little is computed
// on them, so the bytes bound it.  Requests differ in length, so the work is
// cut by tokens and not by requests: the blocks of 128 tokens that the queries
// see, of all requests and KV heads laid end to end, are shared out evenly to
// as many workgroups as the card holds.  A workgroup's share covers parts of a
// few (request, KV head) units; a unit that lies in one share goes straight to
// the output, the others leave a record (running maximum, sum and sum of
// Values) of each part, and a second launch joins them.  Each workgroup finds
// its share from the lengths in device memory, so a captured launch follows
// them.
//
// A wave takes 32 tokens a step.  S^T = K q^T (16 tokens by 16 query heads a
// product) leaves four tokens of one query in each lane, which is how
// O^T = V^T P^T wants them: no weight moves between lanes.  Keys and Values
// come straight from memory in 16-byte pieces; a lane's eight Value rows by
// eight channels are turned by v_perm.  Weights enter the products as two
// 16-bit terms: bf16 leaves 2^-17 of a weight, fp16 2^-23 or, of a weight below
// 2^-9 of the row's largest, 2^-32 of that.
//
// 32 requests of 16000 tokens, 32/8 heads of 128, fp16: 320 us, 6.6 TB/s, where a
// plain read runs at 7.1 (one workgroup a CU 411 and with rows five steps ahead
// 386, of a form of two that took 373).  One of 2400 tokens: 8 us, three memory
// latencies behind each other (length, table, rows), and 4 for the join.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>

#include "rk_paged_dev.h"

namespace {

using rk::base_of;
using rk::f32x4;
using rk::kNone;
using rk::kPagedThreads;
using rk::kPagedWaves;
using rk::PagedArgs;

constexpr int kStep = 32;                     // tokens of a wave's step
constexpr int kBlock = kStep * kPagedWaves;  // tokens of a piece of work
constexpr int kRows = 16;                     // queries of a unit
// Pieces of a unit up to which a workgroup may take all of it: one launch instead of
// two and no records, but the longest unit ends last.
constexpr int kMostAlone = 16;
constexpr int kAloneWaves = 8;  // of such a workgroup, where each CU has one at most
// Waves that join a query of many records (one wave reads four at a time): one text
// of 32000 tokens, 8 query heads to its KV head: 31.3 us in all with 4, 17.8 with 16;
// 8 records a row: 12.9 with one wave, 11.3 with 16, 4 records as long.
constexpr int kJoinWaves = 16;

constexpr float kAlike = 0x1p-14f;  // weight of tokens whose Values only have to show what is not finite

// Pieces of one request and KV head.
__device__ __forceinline__ int pieces_of(const PagedArgs& a, int b) {
  const int p = a.map.pages > 0 ? rk::len_of(a.map, b) - 1 : -1;
  const rk::Seen<kStep> s(max(p, 0), p, a.window, a.sinks);
  return (s.blocks + kPagedWaves - 1) / kPagedWaves;
}

// Shares: workers that get any work, and where share w begins.
struct Shares {
  int64_t pieces;
  int workers;
  __device__ __forceinline__ int64_t begin(int w) const { return w * pieces / workers; }
  __device__ __forceinline__ int of(int64_t piece) const { return (int)(((piece + 1) * workers - 1) / pieces); }
};
__device__ __forceinline__ Shares shares_of(const PagedArgs& a, int per_request, int units) {
  Shares s;
  s.pieces = (int64_t)per_request * units;
  s.workers = (int)min((int64_t)a.workers, s.pieces);
  return s;
}

// Bytes that are used once.
template <class V>
__device__ __forceinline__ V load_once(const void* p) {
  return __builtin_nontemporal_load((const V*)p);
}

// The largest over the four lanes n, 16 + n, 32 + n, 48 + n.
__device__ __forceinline__ float column_max(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  x = fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
  u = __builtin_bit_cast(uint32_t, x);
  const auto t = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t t0 = t[0], t1 = t[1];
  return fmaxf(__builtin_bit_cast(float, t0), __builtin_bit_cast(float, t1));
}

// Pages of a wave's 32 tokens.  Lane (g, n) has Keys of tokens n and 16 + n,
// channels 32 c + 8 g, and Values of tokens 4 g + 0..3 and 16 + 4 g + 0..3,
// channels VC n.  Sixteen neighbouring tokens lie in one page, unless pages have
// eight rows.
struct Pages {
  uint32_t k[2], v[2];
};

// Workgroups of a CU: what their registers allow.
constexpr int per_cu(int KF) { return KF == 4 ? 2 : 3; }

// KF: blocks of 32 channels (2 or 4).  EIGHT: pages of eight rows.  W: waves; more
// than kPagedWaves of them for a unit each alone.
template <class DT, int KF, bool EIGHT, int W>
__global__ __launch_bounds__(64 * W, W == kPagedWaves ? per_cu(KF) : 2) void paged_split_kernel(const PagedArgs a) {
  constexpr bool kAlone = W != kPagedWaves;
  constexpr int KD = 32 * KF;      // channels, stored ones up to D
  constexpr int VC = KD / 16;      // channels of a Value piece: 4 or 8
  constexpr int AccPitch = KD + 4;
  typedef unsigned int piece __attribute__((ext_vector_type(KF)));
  __shared__ int s_wave[kPagedWaves], s_found[2];
  __shared__ float s_acc[W][kRows][AccPitch];
  __shared__ float s_ml[W][kRows][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int blocks = (a.G + kRows - 1) / kRows;
  const int units = a.H * blocks;  // of a request
  auto count = [&](int b) { return pieces_of(a, b); };
  const int w = blockIdx.x;
  Shares sh;
  int64_t at, end, first = 0;  // pieces; the first one of request b
  int b;
  if (kAlone || a.direct) {  // a unit each
    b = w / units;
    const int unit = w - b * units, pieces = pieces_of(a, b);
    at = (int64_t)unit * pieces;
    end = at + pieces;
    if (pieces == 0) {
      const int h = unit / blocks, row0 = (unit - h * blocks) * kRows;
      for (int r = wave; r < min(a.G - row0, kRows); r += W)
        for (int c = lane; c < a.D; c += 64)
          ((uint16_t*)a.out)[b * a.o_sb + (int64_t)(h * a.G + row0 + r) * a.o_sh + c * a.o_sd] = 0;
    }
  } else {
    rk::Line<decltype(count)> line(a.map.B, count, s_wave, s_found);
    sh = shares_of(a, line.total, units);
    if (w >= sh.workers) return;
    at = sh.begin(w);
    end = sh.begin(w + 1);
    const rk::Found found = line.find((int)(at / units));
    b = found.b;
    first = (int64_t)found.before * units;
  }
  while (at < end) {
    const int pieces = pieces_of(a, b);
    if (at >= first + (int64_t)pieces * units) {
      first += (int64_t)pieces * units;
      ++b;
      continue;
    }
    const int unit = (int)((at - first) / pieces);
    const int off = (int)(at - first) - unit * pieces;
    const int take = (int)min((int64_t)(pieces - off), end - at);
    at += take;
    // ---- one part of a unit
    const int h = unit / blocks, row0 = (unit - h * blocks) * kRows;
    const int rows = min(a.G - row0, kRows);
    const int len = rk::len_of(a.map, b), p = len - 1;
    const rk::Seen<kStep> seen(p, p, a.window, a.sinks);
    uint4 q[KF];
    {
      const int64_t qo = b * a.q_sb + (int64_t)(h * a.G + row0 + n) * a.q_sh;
#pragma unroll
      for (int c = 0; c < KF; ++c) {
        const int ch = 32 * c + 8 * g;
        q[c] = make_uint4(0, 0, 0, 0);
        if (n < rows && ch < a.D) {
          const uint16_t* src = (const uint16_t*)a.q + qo + ch * a.q_sd;
          q[c] = a.q_vec ? rk::load8<true>(src, 1, 8) : rk::load8<false>(src, a.q_sd, 8);
        }
      }
    }
    const uint16_t* kb = (const uint16_t*)a.k + h * a.k_sh;
    const uint16_t* vb = (const uint16_t*)a.v + h * a.v_sh;
    float m = kNone, l = 0.f;
    f32x4 acc[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int last = min(kPagedWaves * (off + take), seen.blocks);
    const uint32_t in_page = (1u << a.map.shift) - 1;
    // Bytes from a row group's first row to this lane's piece.  Behind the last
    // token its row is read again, and channels past D are the first ones again:
    // they count for nothing (`part`).
    uint32_t k_off[2], v_off[2][4];
    auto offsets = [&](int left) {  // tokens of the step that are there
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int end = max(left - 16 * s, 1) - 1;
        const uint32_t row = EIGHT ? 0 : min(n, end);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t at = (EIGHT ? min(4 * g + e, end) - min(4 * g, end) : min(4 * g + e, end));
          v_off[s][e] = 2 * (at * (uint32_t)a.v_ss + (VC * n < a.D ? VC * n : 0));
        }
        k_off[s] = 2 * (row * (uint32_t)a.k_ss);
      }
    };
    offsets(kStep);
    auto pages_at = [&](int i) {  // (past the last step: the last one's again)
      const int t0 = seen.token(min(i, last - 1));
      Pages x;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        x.k[s] = rk::page_of(a.map, b, min(t0 + 16 * s + (EIGHT ? n : 0), p));
        x.v[s] = EIGHT ? rk::page_of(a.map, b, min(t0 + 16 * s + 4 * g, p)) : 0;
      }
      return x;
    };
    // The tokens of step i that the queries see and that have a page.
    auto there_of = [&](int i, const Pages& at) {
      const int t0 = seen.token(i);
      uint32_t there = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bool ok = at.k[s] < (uint32_t)a.map.pages && rk::sees(p, t0 + 16 * s + n, a.window, a.sinks);
        there |= (uint32_t)(__ballot(ok) & 0xffff) << (16 * s);
      }
      return there;
    };
    // First rows of either sixteen tokens (the pool's first row where there is no page).
    auto rows_at = [&](int i, const uint32_t (&page)[2], int first, const uint16_t* src, int64_t sp, int64_t ss,
                       const char* (&at)[2]) {
      const int t0 = seen.token(i);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint32_t pg = page[s];
        if (!EIGHT) pg = (uint32_t)__builtin_amdgcn_readfirstlane((int)pg);
        const bool ok = pg < (uint32_t)a.map.pages;
        const int64_t row = min(t0 + 16 * s + (EIGHT ? first : 0), p) & in_page;
        at[s] = (const char*)(src + (ok ? pg : 0u) * sp + (ok ? row : 0) * ss);
      }
    };
    rk::u32x4 k[2][KF];
    uint32_t v[8][KF];
    auto load_k = [&](int i, const Pages& x) {
      const char* at[2];
      rows_at(i, x.k, n, kb, a.k_sp, a.k_ss, at);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int c = 0; c < KF; ++c) {
          const int ch = 32 * c + 8 * g;
          k[s][c] = load_once<rk::u32x4>(at[s] + k_off[s] + 2 * (KD == a.D || ch < a.D ? ch : 0));
        }
    };
    auto load_v = [&](int i, const Pages& x) {
      const char* at[2];
      rows_at(i, EIGHT ? x.v : x.k, 4 * g, vb, a.v_sp, a.v_ss, at);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const piece y = load_once<piece>(at[s] + v_off[s][e]);
#pragma unroll
          for (int d = 0; d < KF; ++d) v[4 * s + e][d] = y[d];
        }
    };
    // Scores of the step whose Keys are there.
    auto score = [&](f32x4 (&sc)[2]) {
#pragma unroll
      for (int c = 0; c < KF; ++c)
        if (32 * c + 32 > a.D) {
#pragma unroll
          for (int s = 0; s < 2; ++s)
            if (32 * c + 8 * g >= a.D) k[s][c] = rk::u32x4{0, 0, 0, 0};
        }
#pragma unroll
      for (int s = 0; s < 2; ++s) sc[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KF; ++c)
#pragma unroll
        for (int s = 0; s < 2; ++s) sc[s] = DT::mfma(__builtin_bit_cast(uint4, k[s][c]), q[c], sc[s]);
    };
    // Nothing of the tokens that are not there: scores -inf, Values zero.
    auto only = [&](uint32_t there, f32x4 (&sc)[2]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool on = there >> (16 * (e >> 2) + 4 * g + (e & 3)) & 1;
        sc[e >> 2][e & 3] = on ? sc[e >> 2][e & 3] : kNone;
#pragma unroll
        for (int d = 0; d < KF; ++d) v[e][d] = on ? v[e][d] : 0;
      }
    };
    // Channels VC n + j of the step's Values, eight tokens.
    auto turned = [&](int j) {
      uint32_t t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        t[e] = j & 1 ? rk::pack_hi(v[2 * e][j >> 1], v[2 * e + 1][j >> 1])
                     : rk::pack_lo(v[2 * e][j >> 1], v[2 * e + 1][j >> 1]);
      return make_uint4(t[0], t[1], t[2], t[3]);
    };
    // As soon as a step's Keys (Values) have been used, their registers take the
    // next step's; the page numbers of the one behind it are on their way too.
    const int i0 = kPagedWaves * off + wave;
    if (i0 < last) {
      auto cut = [&](int i) {  // the step that tokens end in is the last one
        if (seen.token(i) + kStep - 1 > p) {
          asm volatile("");
          offsets(p + 1 - seen.token(i));
        }
      };
      Pages now = pages_at(i0), next = pages_at(i0 + W);
      cut(i0);
      load_k(i0, now);
      load_v(i0, now);
      for (int i = i0; i < last; i += W) {
        const int then = i + W, t0 = seen.token(i);
        // A CU's older workgroup goes first wherever both could, and ends early; by
        // turns they end together (32 requests of 16000 tokens: 344 us, 338 so).
        if (((i / W) ^ (2 * blockIdx.x >= gridDim.x ? 1 : 0)) & 1)
          __builtin_amdgcn_s_setprio(2);
        else
          __builtin_amdgcn_s_setprio(0);
        const bool part = t0 + kStep - 1 > p || (p - t0 >= a.window && t0 + kStep > a.sinks) ||
                          !__all(now.k[0] < (uint32_t)a.map.pages && now.k[1] < (uint32_t)a.map.pages);
        uint32_t there = ~0u;
        if (part) {
          asm volatile("");  // a branch: most steps are whole
          there = there_of(i, now);
        }
        f32x4 sc[2];
        score(sc);
        if (then < last) {
          cut(then);
          load_k(then, next);
        }
        if (part) {
          asm volatile("");
          only(there, sc);
        }
        float top = kNone;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, sc[e >> 2][e & 3]);
        top = column_max(top);
        // against an earlier maximum while weights stay below 2^8, as any base gives
        // the same quotient
        if (__any((top - m) * a.scale_log2 > rk::kSlack)) {
          asm volatile("");
          const float m_new = fmaxf(m, top), keep = rk::fast_exp2((m - base_of(m_new)) * a.scale_log2);
          m = m_new;
          l *= keep;
#pragma unroll
          for (int j = 0; j < VC; ++j) acc[j] *= keep;
        }
        float base = base_of(m) * a.scale_log2;
        if (__any(fabsf(base) > rk::kFar)) {
          asm volatile("");
#pragma unroll
          for (int s = 0; s < 2; ++s) sc[s] -= base_of(m);
          base = 0.f;
        }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = rk::fast_exp2(__builtin_fmaf(sc[e >> 2][e & 3], a.scale_log2, rk::kLift<DT> - base));
          l += x[e];
        }
        uint4 hi, lo;
        DT::split8(x, hi, lo);
#pragma unroll
        for (int j = 0; j < VC; ++j) {
          const uint4 vt = turned(j);
          acc[j] = DT::mfma(vt, hi, acc[j]);
          acc[j] = DT::mfma(vt, lo, acc[j]);
        }
        if (then < last) load_v(then, next);
        now = next;
        next = pages_at(then + W);
      }
    }
    l += rk::shfl_xor(l, 16);
    l += rk::shfl_xor(l, 32);
    // A weight is above zero, and an infinity or a NaN times it is one.  Its two terms are
    // not both: the second is often zero or below, and both are zero where 16 bits hold no
    // less.  So channels that are not finite are summed again with all weights alike, and
    // become what that gives (rows whose sum of weights is NaN are all NaN anyhow): 32
    // requests of 16000 tokens take 385 us with one infinity, 620 where all are, 321
    // without; one request of 2400 tokens 11.5, and 11.1 if it were not looked for.
    bool odd = false;
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) odd |= !(fabsf(acc[j][i]) < __builtin_inff());
    if (__any(odd)) {
      f32x4 kind[VC];
#pragma unroll
      for (int j = 0; j < VC; ++j) kind[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      offsets(kStep);
      for (int i = i0; i < last; i += W) {
        const Pages now = pages_at(i);
        if (seen.token(i) + kStep - 1 > p) offsets(p + 1 - seen.token(i));
        load_k(i, now);
        load_v(i, now);
        const uint32_t there = there_of(i, now);
        f32x4 sc[2];
        score(sc);
        only(there, sc);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = sc[e >> 2][e & 3] == kNone ? 0.f : kAlike;
        uint4 hi, lo;
        DT::split8(x, hi, lo);
#pragma unroll
        for (int j = 0; j < VC; ++j) kind[j] = DT::mfma(turned(j), hi, kind[j]);
      }
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(fabsf(acc[j][i]) < __builtin_inff()) && !(fabsf(kind[j][i]) < __builtin_inff())) acc[j][i] = kind[j][i];
    }
    // ---- the waves' parts: lane (g, n) holds channels VC (4 g + i) + j of query n
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VC; ++j) s_acc[wave][n][VC * (4 * g + i) + j] = acc[j][i];
    if (g == 0) {
      s_ml[wave][n][0] = m * a.scale_log2;
      s_ml[wave][n][1] = l;
    }
    __syncthreads();
    const int r = threadIdx.x >> 4, c0 = VC * n;
    if (r < rows) {
      float top = kNone;
#pragma unroll
      for (int v = 0; v < W; ++v) top = fmaxf(top, s_ml[v][r][0]);
      float sum = 0.f, o[VC];
#pragma unroll
      for (int e = 0; e < VC; ++e) o[e] = 0.f;
#pragma unroll
      for (int v = 0; v < W; ++v) {
        const float f = rk::fast_exp2(s_ml[v][r][0] - base_of(top));
        sum += f * s_ml[v][r][1];
#pragma unroll
        for (int e = 0; e < VC; ++e) o[e] += f * s_acc[v][r][c0 + e];
      }
      if (kAlone || take == pieces) {
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        uint16_t* dst = (uint16_t*)a.out + b * a.o_sb + (int64_t)(h * a.G + row0 + r) * a.o_sh;
#pragma unroll
        for (int e = 0; e < VC; ++e)
          if (c0 + e < a.D) dst[(c0 + e) * a.o_sd] = DT::from_f32(o[e] * inv);
      } else {
        const int64_t rec = ((int64_t)w * 2 + (off > 0 ? 0 : 1)) * kRows + r;
        float* dst = a.acc + rec * KD + c0;
#pragma unroll
        for (int e = 0; e < VC; e += 4) *(float4*)(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        if (n == 0) *(float2*)(a.ml + 2 * rec) = make_float2(top, sum);
      }
    }
    // the shares that the unit lies in, for the launch that joins them
    if (!kAlone && !a.direct && off == 0 && threadIdx.x == 0) {
      const int64_t begin = at - take;
      a.span[b * units + unit] = make_int2(w, sh.of(begin + pieces - 1));
    }
    __syncthreads();
  }
}

// Joins the records of a query, by W waves, or clears it where it sees nothing: four
// queries a workgroup, or one of many records.
template <class DT, int KF, int W>
__global__ __launch_bounds__(W == 1 ? kPagedThreads : 64 * W) void paged_join_kernel(const PagedArgs a) {
  constexpr int KD = 32 * KF;
  constexpr int C = KD / 64;  // channels of a lane
  constexpr int kAhead = 4;
  __shared__ float s_acc[W][KD], s_ml[W][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = W == 1 ? 0 : wave;
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * kPagedWaves + wave : blockIdx.x;
  const bool mine = row < a.N * a.Hq;
  const int b = mine ? (int)(row / a.Hq) : 0, hq = mine ? (int)(row - (int64_t)b * a.Hq) : 0;
  const int h = hq / a.G, r = hq - h * a.G;
  const int blocks = (a.G + kRows - 1) / kRows;
  const int2 span = a.span[(int64_t)b * a.H * blocks + h * blocks + r / kRows];  // (not written where there is nothing)
  const bool none = pieces_of(a, b) == 0;
  if (W == 1 && !mine) return;
  if (!none && span.x == span.y) return;  // the split launch wrote it (all waves of a row)
  uint16_t* dst = (uint16_t*)a.out + b * a.o_sb + (int64_t)hq * a.o_sh;
  const int c0 = C * lane;
  if (none) {
    if (part == 0)
#pragma unroll
      for (int e = 0; e < C; ++e)
        if (c0 + e < a.D) dst[(c0 + e) * a.o_sd] = 0;
    return;
  }
  float m = kNone, l = 0.f, o[C];
#pragma unroll
  for (int e = 0; e < C; ++e) o[e] = 0.f;
  for (int w0 = span.x + part; w0 <= span.y; w0 += W * kAhead) {
    float2 ml[kAhead];
    float x[kAhead][C];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int w = min(w0 + k * W, span.y);
      const int64_t rec = ((int64_t)w * 2 + (w == span.x ? 1 : 0)) * kRows + (r & (kRows - 1));
      ml[k] = *(const float2*)(a.ml + 2 * rec);
#pragma unroll
      for (int e = 0; e < C; ++e) x[k][e] = a.acc[rec * KD + c0 + e];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (w0 + k * W > span.y) break;
      const float top = fmaxf(m, ml[k].x), base = base_of(top);
      const float f0 = rk::fast_exp2(m - base), f1 = rk::fast_exp2(ml[k].x - base);
      l = l * f0 + ml[k].y * f1;
#pragma unroll
      for (int e = 0; e < C; ++e) o[e] = o[e] * f0 + x[k][e] * f1;
      m = top;
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < C; ++e) s_acc[wave][c0 + e] = o[e];
    if (lane == 0) {
      s_ml[wave][0] = m;
      s_ml[wave][1] = l;
    }
    __syncthreads();
    if (wave) return;
    float top = kNone;
#pragma unroll
    for (int i = 0; i < W; ++i) top = fmaxf(top, s_ml[i][0]);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < C; ++e) o[e] = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float f = rk::fast_exp2(s_ml[i][0] - base_of(top));
      l += f * s_ml[i][1];
#pragma unroll
      for (int e = 0; e < C; ++e) o[e] += f * s_acc[i][c0 + e];
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < C; ++e)
    if (c0 + e < a.D) dst[(c0 + e) * a.o_sd] = DT::from_f32(o[e] * inv);
}

// ------------------------------------------------------------------- host
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Pieces of the longest request that a table reaches.
int64_t pieces_of_longest(int64_t cap, int64_t window, int64_t sinks) {
  const int64_t seen = cdiv(std::min(window, cap), kStep) + 1 + cdiv(std::min(sinks, cap), kStep);
  return cdiv(std::min(cdiv(cap, kStep), seen), kPagedWaves);
}

struct Call {
  const rk_tensor *q, *out;
  const rk_pages* pages;        // or
  const rk_tensor *k, *v;       // plain rows, with
  const int32_t* lens;          // their lengths
  const int32_t* starts;
  int64_t groups, window, sinks;
};

struct Plan {
  int64_t B, rows;         // requests; output rows (new tokens times query heads)
  bool single;             // one new token a request
  size_t acc, ml, span, total;  // workspace
  int join;                     // waves that join a row
};

// Checks a call and forms its arguments and workspace; no HIP calls.
int make_plan(const Call& c, int cus, PagedArgs* a, Plan* p) {
  memset(a, 0, sizeof(*a));
  memset(p, 0, sizeof(*p));
  int st;
  const bool plain = c.pages == nullptr;
  if (!c.q || (plain && (!c.k || !c.v))) return RK_ERR_NULL;
  const int rank = plain ? 4 : 3;
  if ((st = rk::check_desc(c.q, rank))) return st;
  const rk_tensor *k = plain ? c.k : &c.pages->k, *v = plain ? c.v : &c.pages->v;
  int64_t cap = 0;
  if (plain) {
    if ((st = rk::check_desc(k, 4)) || (st = rk::check_desc(v, 4))) return st;
    for (int i = 0; i < 4; ++i)
      if (k->shape[i] != v->shape[i]) return RK_ERR_SHAPE;
    if (k->shape[0] != c.q->shape[0]) return RK_ERR_SHAPE;
    cap = k->shape[2];
    if (cap >= (INT64_C(1) << 30) || k->shape[0] >= (INT64_C(1) << 31)) return RK_ERR_SHAPE;
    p->B = k->shape[0];
    a->map.lens = c.lens;
    a->map.B = a->map.pages = (int32_t)p->B;
    a->map.per = 1;
    a->map.shift = 31;
    a->map.cap = (int32_t)cap;
  } else {
    if ((st = rk::set_pages(c.pages, &a->map, &p->B, &cap))) return st;
    if (cap >= (INT64_C(1) << 30)) return RK_ERR_SHAPE;
    if (!c.starts && c.q->shape[0] != p->B) return RK_ERR_SHAPE;
  }
  a->map.starts = c.starts;
  if (!rk::is_half(c.q->dtype) || k->dtype != c.q->dtype || v->dtype != c.q->dtype) return RK_ERR_DTYPE;
  const int64_t D = c.q->shape[rank - 1], Hq = c.q->shape[1], H = k->shape[1];
  if (D < 8 || D > 128 || D % 8 || k->shape[3] != D) return RK_ERR_HEAD_DIM;
  if (c.groups < 1 || H < 1 || H > (1 << 20) || c.groups > (1 << 20) || Hq != H * c.groups) return RK_ERR_HEADS;
  if (!rk::vec_ok(k) || !rk::vec_ok(v)) return RK_ERR_STRIDE;
  // sixteen rows, as the decode's offsets reach, within 32 bits of bytes
  if (k->stride[2] >= (INT64_C(1) << 27) || v->stride[2] >= (INT64_C(1) << 27)) return RK_ERR_STRIDE;
  if (c.window < 0 || c.sinks < 0) return RK_ERR_ARG;
  if (c.out) {
    if ((st = rk::check_desc(c.out, rank))) return st;
    if (c.out->dtype != c.q->dtype) return RK_ERR_DTYPE;
    for (int i = 0; i < rank; ++i) {
      if (c.out->shape[i] != c.q->shape[i]) return RK_ERR_SHAPE;
      if (c.out->shape[i] > 1 && c.out->stride[i] == 0) return RK_ERR_STRIDE;
    }
  }
  const int64_t T = plain ? c.q->shape[2] : c.starts ? 0 : 1;
  const int64_t N = plain ? p->B * T : c.q->shape[0];
  if (T >= (INT64_C(1) << 30) || N >= (INT64_C(1) << 31)) return RK_ERR_SHAPE;
  p->rows = N * Hq;
  p->single = T == 1;
  if (p->rows >= (INT64_C(1) << 30)) return RK_ERR_SHAPE;
  a->map.each = (int32_t)T;
  a->N = N;
  a->T = (int32_t)T;
  a->Hq = (int32_t)Hq; a->H = (int32_t)H; a->G = (int32_t)c.groups; a->D = (int32_t)D;
  a->window = c.window == 0 || c.window > INT_MAX ? INT_MAX : (int32_t)c.window;
  a->sinks = (int32_t)std::min<int64_t>(c.sinks, INT_MAX);
  a->scale_log2 = rk::kLog2e / sqrtf((float)D);
  auto q_strides = [&](const rk_tensor* t, int64_t* sb, int64_t* st_, int64_t* sh, int64_t* sd) {
    *sh = t->stride[1];
    *sb = c.starts ? 0 : t->stride[0];
    *st_ = plain ? t->stride[2] : t->stride[0];
    *sd = t->stride[rank - 1];
  };
  a->q = c.q->data;
  q_strides(c.q, &a->q_sb, &a->q_st, &a->q_sh, &a->q_sd);
  a->q_vec = rk::vec_ok(c.q);
  if (c.out) {
    a->out = c.out->data;
    q_strides(c.out, &a->o_sb, &a->o_st, &a->o_sh, &a->o_sd);
    a->o_vec = rk::vec_ok(c.out);
  }
  a->k = k->data;
  a->k_sp = k->stride[0]; a->k_sh = k->stride[1]; a->k_ss = k->stride[2];
  a->v = v->data;
  a->v_sp = v->stride[0]; a->v_sh = v->stride[1]; a->v_ss = v->stride[2];
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return here;
  };
  if (p->single) {
    const int64_t KD = D <= 64 ? 64 : 128;
    const int64_t units = p->B * H * cdiv(c.groups, kRows), longest = pieces_of_longest(a->map.cap, a->window, a->sinks);
    if (units * (cdiv(cap, kBlock) + 1) >= (INT64_C(1) << 31)) return RK_ERR_SHAPE;
    if (units >= rk::kMostGroups || cdiv(p->rows, kPagedWaves) >= rk::kMostGroups) return RK_ERR_SHAPE;
    // A unit to a workgroup, or all of them shared out evenly with a join.  The first
    // saves the join, its records and the search for shares, 5 us.  A piece of the
    // longest unit takes it 1.85 us with eight waves, where each CU has one unit at most,
    // and 4.3 with four, where units begin at once (128 channels; 1.1 and 2.6 with 64):
    // the memory's latency, a step of a wave each.  All CUs together read a piece of as
    // many units as CUs in 2.5 us (1.4), which bounds either form and is all that the
    // shared one takes.  32 query heads on 8 KV heads of 128, alone and shared: 4 requests
    // of 364 tokens 11.6 and 12.5 us, of 1004 21.2 and 12.9; 16 of 876 20.3 and 20.3; 32 of
    // 2028 46.0 and 49.5; 40 of 492 23.5 and 27.3, of 2028 73.9 and 61.2.  Heads of 64: 4
    // of 1004 13.4 and 10.7, 16 of them 14.6 and 16.7, 40 of them 24.7 and 25.2.  Where
    // requests differ the first gains: 96 of 10 to 1004 47 and 58.
    const bool narrow = D <= 64;
    const double share = (double)units / cus;
    const double all = (narrow ? 1.4 : 2.5) * share;
    const double own = share <= 1 ? (narrow ? 1.1 : 1.85)
                                  : (narrow ? 2.6 : 4.3) * std::max(1.0, share / per_cu(narrow ? 2 : 4));
    const bool alone = longest <= kMostAlone && (double)longest * (std::max(own, all) - all) <= 5.0;
    const int64_t fullest = cdiv(units, cus);
    a->direct = !alone ? 0 : fullest > 1 ? kPagedWaves : kAloneWaves;
    a->workers = (int32_t)(a->direct ? units : std::max<int64_t>(
        std::min<int64_t>(per_cu(D <= 64 ? 2 : 4) * (int64_t)cus, units * longest), 1));
    if (!a->direct) {
      const size_t records = (size_t)a->workers * 2 * kRows;
      p->acc = take(records * KD * 4);
      p->ml = take(records * 8);
      p->span = take((size_t)units * 8);
      // records of a unit, where requests are of one length
      p->join = a->workers > 4 * units ? kJoinWaves : 1;
    }
  } else if (p->rows > 0) {
    // Cut the tokens where the rows alone leave CUs empty.  A part saves its share
    // of the tiles, about a microsecond each, and costs its records, written and
    // read: the two are equal at the square root (3 x 77 queries on 1077 tokens, 8
    // heads of 80: 18.9 us in 4 parts, 16.7 in 6, 17.7 in 9, 20.5 in 17; 512 on 8000,
    // 32/8 heads of 128: 30.3 us whole with a window of 1024, 33.3 in 3).
    const int64_t grid = rk::window_slots(*a) * H;
    const int64_t seen = std::min(cap, std::min<int64_t>(a->window, cap) + std::min<int64_t>(a->sinks, cap) + 128 / c.groups);
    const double tiles = seen / 64.0, record = (double)p->rows * cdiv(D, 32) * 128 * 2 / 3.1e6;
    const int64_t most = std::min(2 * (int64_t)cus / std::max<int64_t>(grid, 1), cdiv(seen, 128));
    a->splits = (int32_t)std::max<int64_t>(std::min<int64_t>(most, (int64_t)sqrt(tiles / record)), 1);
    if (grid * a->splits >= rk::kMostGroups) return RK_ERR_SHAPE;
    // One round, of more than a workgroup a CU: long and short ones on each (causal, 3 x
    // 1018 tokens, 16 query heads to each of 2 of 64: 40.8 us, 29.8 so; 8 x 600, 8 heads
    // of 128: 27.5 and 25.1; requests of equal windows: as long).  More rounds even out by
    // themselves, and keep a request's tiles together.
    if (grid * a->splits > cus && grid * a->splits <= rk::window_per_cu(*a) * cus)
      a->round = (int32_t)std::max<int64_t>(cus / H, 1);
    if (a->splits > 1) {
      p->acc = take((size_t)p->rows * a->splits * cdiv(D, 32) * 128);
      p->ml = take((size_t)p->rows * a->splits * 8);
    }
  }
  p->total = at;
  return RK_OK;
}

int null_data(const Call& c, const PagedArgs& a) {
  if (!a.q || !a.out) return RK_ERR_NULL;
  if (a.map.pages > 0 && a.map.cap > 0 && (!a.k || !a.v)) return RK_ERR_NULL;
  if (c.pages && (!a.map.lens || (a.map.cap > 0 && !a.map.table))) return RK_ERR_NULL;
  return RK_OK;
}

int resolve_cus(int num_cus, int* st) {
  *st = RK_OK;
  if (num_cus > 0) return num_cus;
  const int cus = num_cus < 0 ? 0 : rk::current_device_cus(nullptr);
  if (cus <= 0) *st = num_cus < 0 ? RK_ERR_ARG : RK_ERR_NO_DEVICE;
  return cus;
}

template <class F>
int by_shape(int dtype, int D, F&& f) {
  auto on = [&](auto dt) { D <= 64 ? f(dt, std::integral_constant<int, 2>{}) : f(dt, std::integral_constant<int, 4>{}); };
  dtype == RK_F16 ? on(rk::F16{}) : on(rk::BF16{});
  return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_HIP;
}

int run(const Call& c, void* workspace, size_t workspace_bytes, void* stream) {
  PagedArgs a;
  Plan p;
  // everything but the split is checked before a device is asked for
  int st = make_plan(c, 1, &a, &p);
  if (st) return st;
  if (!c.out) return RK_ERR_NULL;
  if (p.rows == 0 || p.B == 0) return RK_OK;
  if ((st = null_data(c, a))) return st;
  const int cus = resolve_cus(0, &st);
  if (st) return st;
  if ((st = make_plan(c, cus, &a, &p))) return st;
  if (p.total && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < p.total)) return RK_ERR_WORKSPACE;
  a.acc = (float*)((char*)workspace + p.acc);
  a.ml = (float*)((char*)workspace + p.ml);
  a.span = (int2*)((char*)workspace + p.span);
  const hipStream_t s = (hipStream_t)stream;
  if (!p.single) return rk::window_launch(a, c.q->dtype, s);
  return by_shape(c.q->dtype, a.D, [&](auto dt, auto kf) {
    const auto split = [&](auto w) {
      constexpr int W = decltype(w)::value;
      if (a.map.shift == 3)
        hipLaunchKernelGGL((paged_split_kernel<decltype(dt), decltype(kf)::value, true, W>), dim3((unsigned)a.workers),
                           dim3(64 * W), 0, s, a);
      else
        hipLaunchKernelGGL((paged_split_kernel<decltype(dt), decltype(kf)::value, false, W>), dim3((unsigned)a.workers),
                           dim3(64 * W), 0, s, a);
    };
    if (a.direct == kAloneWaves)
      split(std::integral_constant<int, kAloneWaves>{});
    else
      split(std::integral_constant<int, kPagedWaves>{});
    if (a.direct) return;
    if (p.join == 1)
      hipLaunchKernelGGL((paged_join_kernel<decltype(dt), decltype(kf)::value, 1>),
                         dim3((unsigned)cdiv(p.rows, kPagedWaves)), dim3(kPagedThreads), 0, s, a);
    else
      hipLaunchKernelGGL((paged_join_kernel<decltype(dt), decltype(kf)::value, kJoinWaves>), dim3((unsigned)p.rows),
                         dim3(64 * kJoinWaves), 0, s, a);
  });
}

int check_call(const Call& c, int32_t num_cus, size_t* bytes) {
  PagedArgs a;
  Plan p;
  int st = make_plan(c, 1, &a, &p);
  if (st) return st;
  const int cus = resolve_cus(num_cus, &st);
  if (st) return st;
  if ((st = make_plan(c, cus, &a, &p))) return st;
  if (bytes) *bytes = p.total;
  return RK_OK;
}

}  // namespace

extern "C" int rk_paged_attention_check(const rk_tensor* q, const int32_t* starts, const rk_pages* pages,
                                        int64_t num_kv_groups, int64_t window, int64_t sinks, const rk_tensor* out,
                                        int32_t num_cus, size_t* workspace_bytes) {
  if (!pages) return RK_ERR_NULL;
  return check_call({q, out, pages, nullptr, nullptr, nullptr, starts, num_kv_groups, window, sinks}, num_cus,
                    workspace_bytes);
}

extern "C" int rk_paged_attention(const rk_tensor* q, const int32_t* starts, const rk_pages* pages,
                                  int64_t num_kv_groups, int64_t window, int64_t sinks, const rk_tensor* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (!pages) return RK_ERR_NULL;
  return run({q, out, pages, nullptr, nullptr, nullptr, starts, num_kv_groups, window, sinks}, workspace,
             workspace_bytes, stream);
}

extern "C" int rk_window_attention_check(const rk_tensor* q, const rk_tensor* k, const rk_tensor* v,
                                         const int32_t* lens, int64_t num_kv_groups, int64_t window, int64_t sinks,
                                         const rk_tensor* out, int32_t num_cus, size_t* workspace_bytes) {
  return check_call({q, out, nullptr, k, v, lens, nullptr, num_kv_groups, window, sinks}, num_cus, workspace_bytes);
}

extern "C" int rk_window_attention(const rk_tensor* q, const rk_tensor* k, const rk_tensor* v, const int32_t* lens,
                                   int64_t num_kv_groups, int64_t window, int64_t sinks, const rk_tensor* out,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  return run({q, out, nullptr, k, v, lens, nullptr, num_kv_groups, window, sinks}, workspace, workspace_bytes, stream);
}
