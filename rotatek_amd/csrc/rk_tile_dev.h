// rk_tile_dev.h -- attention over rows that many queries share (MI355X,
// gfx950), included by the per-format units rk_tile_*.hip.
//
// The mathematics and the products are rk_span_dev.h's; the split is another.
// There a workgroup's four waves take different tokens for the same 16
// queries, which suits rows that few queries read.  Where a batch shares its
// prefix, one KV head's rows meet all the batch's queries: here the four waves
// take different queries, 16 each, and the same 64 tokens at a time, staged in
// LDS as 16-bit values.  K and V are then read (and quantised rows widened)
// once for 64 queries, and the waves have nothing to join.
//
// A tile's global loads go to registers while the tile before it is worked on,
// then to LDS.  V^T comes out of LDS by transposing reads (four tokens of one
// channel a lane), so no registers are shuffled.  Pieces of 16 bytes are stored
// at another place of their row for each row, so that the rows that one read
// takes the same piece of lie in different banks.
//
// One tile buffer, one tile ahead and 16 queries a wave leave registers and LDS
// for three workgroups on a CU, which hide each other's barriers and latencies:
// 32 queries a wave, two buffers, or two tiles ahead (two workgroups each) took 6,
// 17 and 16 % longer, both halves of a tile in one softmax (spills) 2 to 14 %,
// eight waves that take half a tile each 10 %.  With more than 64 kept channels the
// rotation's staging (85 KB) leaves one workgroup on a CU, for the full-width span
// as well: 64 fp16 requests of 7 heads behind 32768 tokens take 74 us with 64
// channels kept, 154 with 128, and 82 without a rotation.
//
// What bounds it: issue.  64 requests of 7 heads behind 32768 tokens, 64 channels
// kept: 70 to 74 us with the join (11), 320 TFLOP/s of the formula; a wave issues 26
// matrix and 90 other vector instructions for 32 tokens and reads 24 KB of a tile's
// LDS for 64; the matrix pipes are busy for 47 % of the loop, LDS for about as much,
// and waves wait for their turn for 42 % of their time.  32
// requests of 4 heads behind 16001: 34 us with the join (8.6), 2.2 TB/s.
#pragma once

#include "rk_span_dev.h"

namespace rk {

constexpr int kTileTok = 64;

// A thread's share of a tile: pieces of eight channels, row-major.
template <class F, int KB, int VB>
struct TilePart {
  uint32_t k[KB][F::kw], v[VB / 2][F::kw];
  uint8_t ks[KB], vs[VB / 2];
};

// Where piece p of row r lies: rows of P pieces (P = 4, 8, 16; 16 / P rows fill
// the banks once).
template <int P>
__device__ __forceinline__ int swizzle(int p, int r) {
  return p ^ ((r / (16 / P)) & (P - 1));
}

template <class F, int KB, int VB>
__device__ __forceinline__ void load_tile(const Span& sp, const SpanLane<1>& hd, Rsrc vsc, int D, int t0, int tid,
                                          TilePart<F, KB, VB>& x) {
  constexpr int kEl = F::kMx ? 1 : 2;
  const int last = sp.S - 1 - t0;  // rows past the span are its last row
  constexpr int kPiece = 4 * F::kw;
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    const int id = i * kSpanThreads + tid, r = min(id / (4 * KB), last);
    const int p = id % (4 * KB) * 8 < sp.width ? id % (4 * KB) : 0;
    load_words<F::kw>(hd.k, (uint32_t)r * sp.k_ss * kEl + p * kPiece, (uint32_t)t0 * sp.k_ss * kEl, x.k[i]);
    if constexpr (F::kMx)
      x.ks[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(hd.ksc, (uint32_t)(p >> 2) * sp.ksc_sn + r, t0, 0);
  }
#pragma unroll
  for (int i = 0; i < VB / 2; ++i) {
    const int id = i * kSpanThreads + tid, r = min(id / (2 * VB), last);
    const int p = id % (2 * VB) * 8 < D ? id % (2 * VB) : 0;
    load_words<F::kw>(hd.v, (uint32_t)r * sp.v_ss * kEl + p * kPiece, (uint32_t)t0 * sp.v_ss * kEl, x.v[i]);
    if constexpr (F::kMx)
      x.vs[i] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(vsc, (uint32_t)(p >> 2) * sp.vsc_sn + r, t0, 0);
  }
}

// ... widened, to LDS: K [64][4 KB pieces], swizzled, then V [64][2 VB pieces].
// Channels past the row's are zero, and so are rows past the span (their
// weight is 0, which an infinity would make NaN).
template <class F, int KB, int VB>
__device__ __forceinline__ void store_tile(const Span& sp, int D, int t0, int tid, const TilePart<F, KB, VB>& x,
                                           uint4* k, uint4* v) {
  const int n = sp.S - t0;
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    const int id = i * kSpanThreads + tid, r = id / (4 * KB), p = id % (4 * KB);
    uint4 w = widen8<F>(x.k[i], mx_scale(x.ks[i], 0));
    if (8 * p >= sp.width) w = make_uint4(0, 0, 0, 0);
    k[r * (4 * KB) + swizzle<4 * KB>(p, r)] = w;
  }
#pragma unroll
  for (int i = 0; i < VB / 2; ++i) {
    const int id = i * kSpanThreads + tid, r = id / (2 * VB), p = id % (2 * VB);
    uint4 w = widen8<F>(x.v[i], mx_scale(x.vs[i], 0));
    if (r >= n) w = make_uint4(0, 0, 0, 0);
    v[r * (2 * VB) + swizzle_v<2 * VB>(p, r)] = w;
  }
}

// One chunk of a span for the wave's 16 queries, which pre() leaves in q, off and,
// where it is not the call's, scale.
template <class F, int KB, int VB, int NT, int NP, class Pre>
__device__ __forceinline__ void run_tiles(const SpanArgs& a, const Span& sp, const SpanLane<1>& hd, Rsrc vsc, int chunk,
                                          int tid, char* mem, State<VB>& st, const Pre& pre) {
  using TT = typename F::TT;
  const int lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int first = chunk * sp.chunk, lim = min(first + sp.chunk, sp.S);
  constexpr int kKBytes = kTileTok * 64 * KB;
  TilePart<F, KB, VB> part;
  load_tile<F, KB, VB>(sp, hd, vsc, a.D, first, tid, part);
  uint4 q[NT][KB];
  float off, scale = a.scale_log2;
  pre(q, off, scale);
  __syncthreads();  // (the queries' LDS is the tiles')
  store_tile<F, KB, VB>(sp, a.D, first, tid, part, (uint4*)mem, (uint4*)(mem + kKBytes));
  __syncthreads();
  const uint4* ks = (const uint4*)mem;
  const char* vs = mem + kKBytes;
  for (int t0 = first; t0 < lim; t0 += kTileTok) {
    const bool more = t0 + kTileTok < lim;
    if (more) load_tile<F, KB, VB>(sp, hd, vsc, a.D, t0 + kTileTok, tid, part);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tb = t0 + 32 * h;
      if (tb >= lim) break;
      f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int r = 32 * h + 16 * tt + n;
          const uint4 kop = ks[r * (4 * KB) + swizzle<4 * KB>(4 * j + g, r)];
#pragma unroll
          for (int t = 0; t < NT; ++t) s[tt] = TT::mfma(kop, q[t][j], s[tt]);
        }
      const bool whole = tb + 32 <= lim;
      uint32_t on = 0xffu;
      if (!whole) {
        on = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) on |= (uint32_t)(tb + token_of(g, r) < lim) << r;
      }
      // channel slot j: channels 16 j .. 16 j + 15, one a lane
      auto turn = [&](int w, uint4& lo, uint4& hi) {
        lo = read_columns<2 * VB>(vs, 32 * h, 2 * w, g, n);
        hi = read_columns<2 * VB>(vs, 32 * h, 2 * w + 1, g, n);
      };
      weigh_block<TT, VB, NP, true>(s, scale, off, whole, on, st, turn);
    }
    __syncthreads();
    if (more)
      store_tile<F, KB, VB>(sp, a.D, t0 + kTileTok, tid, part, (uint4*)mem, (uint4*)(mem + kKBytes));
    __syncthreads();
  }
}

template <class F, int KV, int KF, int NT, int NP>
__global__ void __launch_bounds__(kSpanThreads, 3) tile_kernel(const SpanArgs a) {
  using TT = typename F::TT;
  constexpr int VB = KF == 2 ? 4 : 8;
  constexpr int DV = 16 * VB;
  constexpr int NTV = NT < 2 ? 2 : NT;
  constexpr int kRows = 64;
  constexpr int kKB = KV > KF ? KV : KF;
  constexpr int kTiles = kTileTok * (64 * kKB + 32 * VB);
  constexpr int kWide = 32 * KV + 8;
  constexpr int kQ = KV > 0 ? 2 * (NTV * kRows * kWide + kRows * 136 + 128 * 32 * KV + 128) : 0;
  __shared__ __attribute__((aligned(16))) char s_mem[kTiles > kQ ? kTiles : kQ];
  __shared__ float s_bias[KV > 0 ? kRows : 1];
  constexpr bool kScaled = KV > 0 && TT::kRk == F16::kRk;
  __shared__ uint32_t s_qtop[kScaled ? kRows : 1];
  uint16_t* s_q = (uint16_t*)s_mem;
  uint16_t* s_raw = s_q + NTV * kRows * kWide;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int id = (int)blockIdx.x;
  const int k = id >= a.first[kFull] ? kFull : kRotated;
  const Span sp = a.span[k];
  const int rel = id - a.first[k];
  // row blocks of the same rows on one XCD, as in span_kernel
  const int blocks = a.blocks[k], heads = a.heads[k];
  const int q8 = __builtin_amdgcn_readfirstlane((rel >> 3) / blocks);
  const int t = 8 * q8 + (rel & 7), R0 = ((rel >> 3) - q8 * blocks) * kRows;
  const int x = __builtin_amdgcn_readfirstlane(t / heads), kv = t - x * heads;
  if (x >= sp.wgs) return;
  const int rows = min(a.B * a.G - R0, kRows);
  const int r = 16 * wave + n;  // the lane's query
  const RowOf o = row_of(a, true, 0, kv, R0 + min(r, rows - 1));
  const int64_t row = (int64_t)o.b * a.Hq + o.h;

  State<VB> st;
  st.clear();

  // (every row and piece is clamped into the span: the buffers' bounds do not
  // count the scalar offset)
  SpanLane<1> hd;
  Rsrc vsc;
  hd.k = make_rsrc((const char*)sp.k + (F::kMx ? 1 : 2) * (kv * sp.k_sh));
  hd.v = make_rsrc((const char*)sp.v + (F::kMx ? 1 : 2) * (kv * sp.v_sh));
  if constexpr (F::kMx) {
    hd.ksc = make_rsrc(sp.ksc + kv * sp.ksc_sh);
    vsc = make_rsrc(sp.vsc + kv * sp.vsc_sh);
  }
  const bool f16 = F::kMx ? a.q_dtype == F16::kRk : TT::kRk == F16::kRk;

  bool done = false;
  if constexpr (KV > 0) {
    if (k == kRotated) {
      Queries<4, 4> qw;
      Rotation<KV> rot;
      if (!a.qr) {
        load_queries<4, 4>(a, true, 0, kv, R0, rows, tid, qw);
        load_rotation<KV>(a, 0, kv, tid, rot);
      }
      auto pre = [&](uint4(&q)[NTV][KV], float& off, float& scale) {
        if (!a.qr) {
          uint4* s_r = (uint4*)(s_raw + kRows * 136);
          uint4* s_mu = s_r + 128 * 4 * KV;
          stage_queries<TT, 1, 4, 4, 128>(tid, qw, f16, s_raw, 136);
          stage_rotation<KV>(tid, rot, s_r, s_mu);
          if constexpr (kScaled)
            if (tid < kRows) s_qtop[tid] = 0u;
          __syncthreads();
          rotate_queries<TT, NTV, 4, KV>(a, wave, lane, f16, s_raw, s_r, s_mu, s_q, kWide, s_bias, s_qtop);
        }
#pragma unroll
        for (int t = 0; t < NTV; ++t)
#pragma unroll
          for (int j = 0; j < KV; ++j)
            q[t][j] = a.qr ? *(const uint4*)(a.qr + (row * NTV + t) * (32 * KV) + 32 * j + 8 * g)
                           : *(const uint4*)(s_q + (t * kRows + r) * kWide + 32 * j + 8 * g);
        off = (a.qr ? a.bias[row] : s_bias[r]) * a.scale_log2 + kLift<TT>;
        if constexpr (kScaled)
          scale = ldexpf(scale, split_shift(a.qr ? a.qtop[row] : __builtin_bit_cast(float, s_qtop[r])));
      };
      run_tiles<F, KV, VB, NTV, NP>(a, sp, hd, vsc, x, tid, s_mem, st, pre);
      done = true;
    }
  }
  if (!done) {
    auto pre = [&](uint4(&q)[NT][KF], float& off, float&) {
      off = kLift<TT>;
      const uint16_t* src = (const uint16_t*)a.q + o.b * a.q_sb + o.h * a.q_sh;
#pragma unroll
      for (int j = 0; j < KF; ++j) {
        const int c = 32 * j + 8 * g;
        const uint4 w = c < a.D ? *(const uint4*)(src + c) : make_uint4(0, 0, 0, 0);
        if constexpr (NT == 1) {
          q[0][j] = w;
        } else {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint16_t h = (uint16_t)(word(w, e >> 1) >> (16 * (e & 1)));
            v[e] = f16 ? F16::to_f32(h) : BF16::to_f32(h);
          }
          uint4 x2[NT];
          terms8<TT, NT>(v, x2);
#pragma unroll
          for (int t = 0; t < NT; ++t) q[t][j] = x2[t];
        }
      }
    };
    run_tiles<F, KF, VB, NT, NP>(a, sp, hd, vsc, x, tid, s_mem, st, pre);
  }

  // the record, straight from the registers
  const float top = row_max(st.top);
  const bool seen = top > -INFINITY;
  const float M = seen ? top + st.m - kLift<TT> : kNegInit;
  const float f = seen ? fast_exp2(st.m - M - kLift<TT>) : 0.f;
  if (r >= rows) return;
  const int64_t at = row * a.np + sp.np0 + x;
#pragma unroll
  for (int j = 0; j < VB; ++j) *(f32x4*)(a.acc + at * DV + 16 * j + 4 * g) = st.acc[j] * f;
  if (g == 0) *(float2*)(a.ml + 2 * at) = make_float2(M, st.l[0] * f);
}

// Widths as in pick_widths.
template <class F, int NT, int NP>
hipError_t pick_tiles(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s) {
#define RK_TILE(KV, KF)                                                                                \
  if (kv == KV && kf == KF) {                                                                          \
    hipLaunchKernelGGL((tile_kernel<F, KV, KF, NT, NP>), dim3(grid), dim3(kSpanThreads), 0, s, a);     \
    return hipGetLastError();                                                                          \
  }
  RK_TILE(0, 2) RK_TILE(1, 2) RK_TILE(2, 2) RK_TILE(0, 4) RK_TILE(1, 4) RK_TILE(2, 4) RK_TILE(4, 4)
#undef RK_TILE
  return hipErrorInvalidValue;
}

}  // namespace rk
