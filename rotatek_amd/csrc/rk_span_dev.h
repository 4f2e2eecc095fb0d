// rk_span_dev.h -- one token's attention over spans of plain or quantised
// rows (MI355X, gfx950), included by the per-format units rk_span_*.hip.
//
// For a query row r and the tokens t of its spans
//   s_rt = (k_t . q_r + bias_r) log2(e) / sqrt(D),  o_r = sum_t 2^s_rt v_t,
//   l_r = sum_t 2^s_rt,  all under a running maximum m_r;
// a workgroup covers one chunk of one span for one unit of query rows and
// leaves (m, l, o) for each row; merge_rows joins a row's records.
//
// Units.  A unit is up to 16 NR query rows that read the same K and V: the
// heads of a KV group, or, over a span that the batch shares, all the batch's
// queries on a KV head.  Each K/V byte is then read once per 16 NR rows.
//
// A workgroup is four waves that take interleaved blocks of 32 tokens.  Rows
// come straight from memory into registers in the matrix core's layout, so a
// block costs no LDS traffic and no barrier:
//   S^T = K Q^T   v_mfma_f32_16x16x32: A = K, 16 tokens x 32 channels.  A
//                 lane's four-lane-group g holds whole 8-channel pieces, and
//                 any order of channels will do as long as Q has the same;
//   O^T += V^T P^T  A = V^T: a lane holds eight tokens of VB channels as it
//                 loads them and transposes them in registers.  P^T is the
//                 lane's own eight scores: A's rows are dealt so that the
//                 lane (g, n) gets tokens 8g .. 8g + 7 of query n.
// Quantised rows are widened to bf16, which holds code 2^e exactly, by the
// conversion that applies the block's scale; queries then enter as one, two
// or three bf16 terms, in which bf16, fp16 and fp32 are exact.
#pragma once

#include <math.h>

#include "rk_common.h"
#include "rk_span.h"

namespace rk {

// ------------------------------------------------------------ row formats
// kw: 32-bit words of eight channels.  piece(g, j): first channel of the
// lane's j-th eight of a score row of KB blocks.
template <class TT_>
struct PlainFmt {
  using TT = TT_;
  static constexpr bool kMx = false;
  static constexpr int kw = 4;
};
struct Mx8Fmt {
  using TT = BF16;
  static constexpr bool kMx = true;
  static constexpr int kw = 2;
  template <int I>
  static __device__ __forceinline__ uint32_t pair(const uint32_t* w, float sc) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[I >> 1], sc, (I & 1) != 0);
    return __builtin_bit_cast(uint32_t, v);
  }
};
struct Mx4Fmt {
  using TT = BF16;
  static constexpr bool kMx = true;
  static constexpr int kw = 1;
  template <int I>
  static __device__ __forceinline__ uint32_t pair(const uint32_t* w, float sc) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], sc, I);
    return __builtin_bit_cast(uint32_t, v);
  }
};

// A block's scale from its byte: the conversions read the exponent field, 255
// makes NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Eight channels as a matrix operand.
template <class F>
__device__ __forceinline__ uint4 widen8(const uint32_t* w, float sc) {
  if constexpr (F::kMx)
    return make_uint4(F::template pair<0>(w, sc), F::template pair<1>(w, sc), F::template pair<2>(w, sc),
                      F::template pair<3>(w, sc));
  else
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int N>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (N == 4) {
    const u32x4 v = *(const u32x4*)p;
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *(const uint2*)p;
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *(const uint32_t*)p;
  }
}

// A block of 32 tokens as one wave holds it.  k[tt]: the lane's 8 KB channels
// of token 8 (n / 4) + 4 tt + n % 4; v[r]: its VB channels of token 8 g + r.
template <class F, int KB, int VB>
struct Block {
  static constexpr int kvw = VB == 8 ? F::kw : (F::kw + 1) / 2;
  uint32_t k[2][KB * F::kw];
  uint32_t v[8][kvw];
  uint32_t ks[2];
  uint2 vs;
};

struct SpanHead {  // a unit's rows of one span
  const char* k;
  const char* v;
  const uint8_t* ksc;
  const uint8_t* vsc;
};

// Loads block `blk`; rows past the span are its last row.
template <class F, int KB, int VB, bool VEC>
__device__ __forceinline__ void load_block(const Span& sp, const SpanHead& hd, int D, int blk, int g, int n,
                                           Block<F, KB, VB>& x) {
  const uint32_t last = (uint32_t)sp.S - 1;
  const uint32_t t0 = (uint32_t)blk * kSpanBlk;
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    const uint32_t t = min(t0 + 8 * (n >> 2) + 4 * tt + (n & 3), last);
    if constexpr (F::kMx) {
      // eight KB channels in one piece; past the row's width the first ones
      // stand in (the query is zero there)
      const uint32_t c = 8 * KB * g < sp.width ? 8 * KB * g : 0;
      const char* p = hd.k + t * sp.k_ss + (F::kw == 2 ? c : c >> 1);
      constexpr int kAll = KB * F::kw;
      if constexpr (kAll == 8) {
        load_words<4>(p, x.k[tt]);
        load_words<4>(p + 16, x.k[tt] + 4);
      } else {
        load_words<kAll>(p, x.k[tt]);
      }
      x.ks[tt] = hd.ksc[(c >> 5) * sp.ksc_sn + t];
    } else if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < KB; ++j) {
        const int c = 32 * j + 8 * g;
        load_words<4>(hd.k + 2 * (t * sp.k_ss + (uint32_t)(c < sp.width ? c : 0)), x.k[tt] + 4 * j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < KB; ++j) {
        const int c = 32 * j + 8 * g;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t v = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (c + 2 * w + e < sp.width)
              v |= (uint32_t)((const uint16_t*)hd.k)[t * sp.k_ss + (c + 2 * w + e) * sp.k_sd] << (16 * e);
          x.k[tt][4 * j + w] = v;
        }
      }
    }
  }
  const int cv = n * VB < D ? n * VB : 0;  // lanes past the head's channels: any will do
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const uint32_t t = min(t0 + 8 * g + r, last);
    if constexpr (F::kMx) {
      if constexpr (VB == 8)
        load_words<F::kw>(hd.v + t * sp.v_ss + (F::kw == 2 ? cv : cv >> 1), x.v[r]);
      else if constexpr (F::kw == 2)
        load_words<1>(hd.v + t * sp.v_ss + cv, x.v[r]);
      else
        x.v[r][0] = *(const uint16_t*)(hd.v + t * sp.v_ss + (cv >> 1));
    } else if constexpr (VEC) {
      load_words<VB / 2>(hd.v + 2 * (t * sp.v_ss + (uint32_t)cv), x.v[r]);
    } else {
#pragma unroll
      for (int w = 0; w < VB / 2; ++w) {
        uint32_t v = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (cv + 2 * w + e < D)
            v |= (uint32_t)((const uint16_t*)hd.v)[t * sp.v_ss + (cv + 2 * w + e) * sp.v_sd] << (16 * e);
        x.v[r][w] = v;
      }
    }
  }
  // eight tokens' scales of the lane's block column; the column is padded to
  // whole groups of 32
  if constexpr (F::kMx) x.vs = *(const uint2*)(hd.vsc + (cv >> 5) * sp.vsc_sn + min(t0, last & ~31u) + 8 * g);
}

// Values as the products take them: x as the sum of NT 16-bit terms.
template <class TT, int NT>
__device__ __forceinline__ void terms8(const float (&x)[8], uint4 (&o)[NT]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = TT::pack2(r[2 * e], r[2 * e + 1]);
      if (i + 1 < NT) {
        r[2 * e] -= TT::to_f32((uint16_t)w[e]);
        r[2 * e + 1] -= TT::to_f32((uint16_t)(w[e] >> 16));
      }
    }
    o[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// fp16 probabilities are formed as 2^14 p (at most 16384): those below 2^-28,
// not 2^-14, fall into fp16's subnormals.  Sums carry the factor until the
// workgroup's record, which is free of it.
template <class TT>
constexpr float kLift = TT::kRk == 0 ? 14.f : 0.f;

// The running state of one wave: NR blocks of 16 query rows.
template <int NR, int VB>
struct State {
  float m[NR], l[NR];
  f32x4 acc[NR][VB];
};

// One chunk of one span: adds the wave's blocks to `st`.  sq: the unit's
// queries in LDS, [term][row][stride] 16-bit, in the lane's channel order.
template <class F, int KB, int VB, int NR, int NT, int NP, bool VEC>
__device__ __forceinline__ void run_span(const SpanArgs& a, const Span& sp, const SpanHead& hd, int b, int x, int wave,
                                         int lane, const uint16_t* sq, int qstride, const float* sbias,
                                         State<NR, VB>& st) {
  using TT = typename F::TT;
  const int g = lane >> 4, n = lane & 15;
  int lim = min(x * sp.chunk + sp.chunk, sp.S);
  if (sp.len) lim = min(lim, max(sp.len[b], 0));
  const int blk0 = x * sp.chunk / kSpanBlk, nblk = (lim + kSpanBlk - 1) / kSpanBlk;
  constexpr bool kRegQ = NR * NT * KB <= 16;  // queries held in registers
  uint4 qreg[kRegQ ? NR : 1][kRegQ ? NT : 1][kRegQ ? KB : 1];
  auto qload = [&](int nr, int t, int j) {
    const int c = F::kMx ? 8 * KB * g + 8 * j : 32 * j + 8 * g;
    return *(const uint4*)(sq + ((t * NR + nr) * 16 + n) * qstride + c);
  };
  if constexpr (kRegQ) {
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < KB; ++j) qreg[nr][t][j] = qload(nr, t, j);
  }
  float bias[NR];
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) bias[nr] = sbias ? sbias[nr * 16 + n] : 0.f;

  auto compute = [&](const Block<F, KB, VB>& x, int blk) {
    f32x4 s[2][NR];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) s[tt][nr] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KB; ++j)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        uint4 kop = widen8<F>(x.k[tt] + j * F::kw, mx_scale(x.ks[tt]));
        // plain rows narrower than KB blocks: no value of another channel
        // meets the query's zero (an infinity would make NaN)
        if constexpr (!F::kMx && VEC)
          if (sp.width < 32 * KB && 32 * j + 8 * g >= sp.width) kop = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if constexpr (kRegQ)
              s[tt][nr] = TT::mfma(kop, qreg[nr][t][j], s[tt][nr]);
            else
              s[tt][nr] = TT::mfma(kop, qload(nr, t, j), s[tt][nr]);
          }
      }
    // which of the lane's eight tokens count
    const int t0 = blk * kSpanBlk + 8 * g;
    uint32_t on = 0xffu;
    const bool whole = (blk + 1) * kSpanBlk <= lim && !sp.mask;
    if (!whole) {
      on = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        bool ok = t0 + r < lim;
        if (sp.mask && ok) ok = sp.mask[b * sp.m_sb + (t0 + r) * sp.m_ss] != 0;
        on |= (uint32_t)ok << r;
      }
    }
    uint4 p[NR][NP];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      float sc[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        sc[r] = (s[r >> 2][nr][r & 3] + bias[nr]) * a.scale_log2;
        if (!((on >> r) & 1u)) sc[r] = -INFINITY;
      }
      float mx = sc[0];
#pragma unroll
      for (int r = 1; r < 8; ++r) mx = fmaxf(mx, sc[r]);
      mx = fmaxf(mx, shfl_xor(mx, 16));
      mx = fmaxf(mx, shfl_xor(mx, 32));
      const float m_new = fmaxf(st.m[nr], mx);
      const float alpha = fast_exp2(st.m[nr] - m_new);
      if (__any(m_new != st.m[nr])) {
#pragma unroll
        for (int j = 0; j < VB; ++j) st.acc[nr][j] *= alpha;
      }
      st.m[nr] = m_new;
      const float base = m_new - kLift<TT>;
      float ps = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        sc[r] = fast_exp2(sc[r] - base);
        ps += sc[r];
      }
      st.l[nr] = st.l[nr] * alpha + ps;
      terms8<TT, NP>(sc, p[nr]);
    }
    // V^T: eight tokens of channel slot j
    uint32_t vw[8][VB / 2];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (F::kMx) {
        const float sc = mx_scale(((r < 4 ? x.vs.x : x.vs.y) >> (8 * (r & 3))) & 0xffu);
        vw[r][0] = F::template pair<0>(x.v[r], sc);
        vw[r][1] = F::template pair<1>(x.v[r], sc);
        if constexpr (VB == 8) {
          vw[r][2] = F::template pair<2>(x.v[r], sc);
          vw[r][3] = F::template pair<3>(x.v[r], sc);
        }
      } else {
#pragma unroll
        for (int w = 0; w < VB / 2; ++w) vw[r][w] = x.v[r][w];
      }
      // rows that do not count hold anything: 0 x NaN must not reach the sum
      if (!whole) {
        const bool ok = (on >> r) & 1u;
#pragma unroll
        for (int w = 0; w < VB / 2; ++w) vw[r][w] = ok ? vw[r][w] : 0u;
      }
    }
#pragma unroll
    for (int j = 0; j < VB; ++j) {
      const int w = j >> 1;
      uint4 av;
      if (j & 1) {
        av.x = pack_hi(vw[0][w], vw[1][w]); av.y = pack_hi(vw[2][w], vw[3][w]);
        av.z = pack_hi(vw[4][w], vw[5][w]); av.w = pack_hi(vw[6][w], vw[7][w]);
      } else {
        av.x = pack_lo(vw[0][w], vw[1][w]); av.y = pack_lo(vw[2][w], vw[3][w]);
        av.z = pack_lo(vw[4][w], vw[5][w]); av.w = pack_lo(vw[6][w], vw[7][w]);
      }
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int t = 0; t < NP; ++t) st.acc[nr][j] = TT::mfma(av, p[nr][t], st.acc[nr][j]);
    }
  };

  Block<F, KB, VB> blk;
  for (int i = blk0 + wave; i < nblk; i += kSpanWaves) {
    load_block<F, KB, VB, VEC>(sp, hd, a.D, i, g, n, blk);
    compute(blk, i);
  }
}

// Query row r of a unit: its batch row and head.
struct RowOf {
  int b, h;
};
__device__ __forceinline__ RowOf row_of(const SpanArgs& a, bool shared, int b, int kv, int R) {
  RowOf o;
  o.b = shared ? R / a.G : b;
  o.h = kv * a.G + (shared ? R - o.b * a.G : R);
  return o;
}

template <class F, int KV, int KF, int NR, int NT, int NP, bool VEC>
__global__ void __launch_bounds__(kSpanThreads) span_kernel(const SpanArgs a) {
  using TT = typename F::TT;
  constexpr int VB = KF == 2 ? 4 : 8;
  constexpr int DV = 16 * VB;
  constexpr int NTV = NT < 2 ? 2 : NT;  // terms of a rotated query
  constexpr int kRows = 16 * NR;
  constexpr int kWide = 32 * (KV > KF ? KV : KF) + 8;  // +8: rows start in other banks
  constexpr int kQ = kRows * kWide * (KV > 0 ? NTV : NT);
  constexpr int kAcc = 2 * kRows * DV;  // two waves' sums
  __shared__ __attribute__((aligned(16))) char s_mem[kQ * 2 > kAcc * 4 ? kQ * 2 : kAcc * 4];
  __shared__ float s_bias[kRows];
  __shared__ float s_m[kSpanWaves][kRows], s_l[kSpanWaves][kRows];
  uint16_t* s_q = (uint16_t*)s_mem;
  float* s_acc = (float*)s_mem;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int id = (int)blockIdx.x;
  const int k = id >= a.first[2] ? kTail : id >= a.first[1] ? kFull : kRotated;
  const Span& sp = a.span[k];
  const int rel = id - a.first[k];
  const int x = rel / a.units[k], u = rel - x * a.units[k];
  const bool shared = a.shared && k != kTail;
  const int blocks = a.blocks[k];
  const int ukv = u / blocks, R0 = (u - ukv * blocks) * kRows;
  const int b = shared ? 0 : ukv / a.H, kv = shared ? ukv : ukv - b * a.H;
  const int rows = min((shared ? a.B * a.G : a.G) - R0, kRows);

  SpanHead hd;
  constexpr int kEl = F::kMx ? 1 : 2;
  hd.k = (const char*)sp.k + kEl * (b * sp.k_sb + kv * sp.k_sh);
  hd.v = (const char*)sp.v + kEl * (b * sp.v_sb + kv * sp.v_sh);
  if constexpr (F::kMx) {
    hd.ksc = sp.ksc + b * sp.ksc_sb + kv * sp.ksc_sh;
    hd.vsc = sp.vsc + b * sp.vsc_sb + kv * sp.vsc_sh;
  }

  State<NR, VB> st;
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
    st.m[nr] = kNegInit;
    st.l[nr] = 0.f;
#pragma unroll
    for (int j = 0; j < VB; ++j) st.acc[nr][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }

  bool done = false;
  if constexpr (KV > 0) {
    if (k == kRotated) {
      constexpr int W = 32 * KV;
      for (int i = tid; i < NTV * kRows * (W / 8); i += kSpanThreads) {
        const int c = 8 * (i % (W / 8)), r = (i / (W / 8)) % kRows, t = i / (W / 8) / kRows;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows && c < a.Dkp) {
          const RowOf o = row_of(a, shared, b, kv, R0 + r);
          v = *(const uint4*)(a.qr + (((int64_t)o.b * a.Hq + o.h) * NTV + t) * a.Dkp + c);
        }
        *(uint4*)(s_q + (t * kRows + r) * kWide + c) = v;
      }
      for (int r = tid; r < kRows; r += kSpanThreads) {
        float v = 0.f;
        if (r < rows) {
          const RowOf o = row_of(a, shared, b, kv, R0 + r);
          v = a.bias[(int64_t)o.b * a.Hq + o.h];
        }
        s_bias[r] = v;
      }
      __syncthreads();
      run_span<F, KV, VB, NR, NTV, NP, VEC>(a, sp, hd, b, x, wave, lane, s_q, kWide, s_bias, st);
      done = true;
    }
  }
  if (!done) {
    constexpr int W = 32 * KF;
    for (int i = tid; i < kRows * (W / 8); i += kSpanThreads) {
      const int c = 8 * (i % (W / 8)), r = i / (W / 8);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
      if (r < rows) {
        const RowOf o = row_of(a, shared, b, kv, R0 + r);
        const int64_t off = o.b * a.q_sb + o.h * a.q_sh;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < a.D) v[e] = load_any(a.q, off + (c + e) * a.q_sd, a.q_dtype);
      }
      uint4 t[NT];
      terms8<TT, NT>(v, t);
#pragma unroll
      for (int j = 0; j < NT; ++j) *(uint4*)(s_q + (j * kRows + r) * kWide + c) = t[j];
    }
    __syncthreads();
    run_span<F, KF, VB, NR, NT, NP, VEC>(a, sp, hd, b, x, wave, lane, s_q, kWide, nullptr, st);
  }

  // join the four waves: the common maximum, then sums in pairs through LDS
  __syncthreads();
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
    st.l[nr] += shfl_xor(st.l[nr], 16);
    st.l[nr] += shfl_xor(st.l[nr], 32);
    if (g == 0) {
      s_m[wave][16 * nr + n] = st.m[nr];
      s_l[wave][16 * nr + n] = st.l[nr];
    }
  }
  __syncthreads();
  float M[NR], L[NR];
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
    const int r = 16 * nr + n;
    M[nr] = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    L[nr] = 0.f;
#pragma unroll
    for (int w = 0; w < kSpanWaves; ++w) L[nr] += s_l[w][r] * fast_exp2(s_m[w][r] - M[nr] - kLift<TT>);
    const float f = fast_exp2(st.m[nr] - M[nr] - kLift<TT>);
#pragma unroll
    for (int j = 0; j < VB; ++j) st.acc[nr][j] *= f;
  }
  // s_acc[slot][row][channel]; a lane's values of one row are VB neighbours
  auto put = [&](int slot) {
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VB; j += 4)
          *(f32x4*)(s_acc + ((slot * kRows + 16 * nr + n) * DV + (4 * g + i) * VB + j)) =
              (f32x4){st.acc[nr][j][i], st.acc[nr][j + 1][i], st.acc[nr][j + 2][i], st.acc[nr][j + 3][i]};
  };
  auto add = [&](int slot) {
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VB; j += 4) {
          const f32x4 v = *(const f32x4*)(s_acc + ((slot * kRows + 16 * nr + n) * DV + (4 * g + i) * VB + j));
#pragma unroll
          for (int e = 0; e < 4; ++e) st.acc[nr][j + e][i] += v[e];
        }
  };
  if (wave >= 2) put(wave - 2);
  __syncthreads();
  if (wave < 2) add(wave);
  __syncthreads();
  if (wave == 1) put(0);
  __syncthreads();
  if (wave != 0) return;
  add(0);
  const int rec = sp.np0 + x;
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
    const int r = 16 * nr + n;
    if (r >= rows) continue;
    const RowOf o = row_of(a, shared, b, kv, R0 + r);
    const int64_t at = ((int64_t)o.b * a.Hq + o.h) * a.np + rec;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VB; j += 4)
        *(f32x4*)(a.acc + at * DV + (4 * g + i) * VB + j) =
            (f32x4){st.acc[nr][j][i], st.acc[nr][j + 1][i], st.acc[nr][j + 2][i], st.acc[nr][j + 3][i]};
    if (g == 0) *(float2*)(a.ml + 2 * at) = make_float2(M[nr], L[nr]);
  }
}

template <class F, int KV, int KF, int NR, int NT, int NP, bool VEC>
hipError_t launch_span(const SpanArgs& a, unsigned grid, hipStream_t s) {
  hipLaunchKernelGGL((span_kernel<F, KV, KF, NR, NT, NP, VEC>), dim3(grid), dim3(kSpanThreads), 0, s, a);
  return hipGetLastError();
}

// The instantiation for a call's widths and row blocks.
template <class F, int NT, int NP, bool VEC, int NR>
hipError_t pick_widths(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s) {
  if (kf == 2) {
    switch (kv) {
      case 0: return launch_span<F, 0, 2, NR, NT, NP, VEC>(a, grid, s);
      case 1: return launch_span<F, 1, 2, NR, NT, NP, VEC>(a, grid, s);
      default: return launch_span<F, 2, 2, NR, NT, NP, VEC>(a, grid, s);
    }
  }
  switch (kv) {
    case 0: return launch_span<F, 0, 4, NR, NT, NP, VEC>(a, grid, s);
    case 1: return launch_span<F, 1, 4, NR, NT, NP, VEC>(a, grid, s);
    case 2: return launch_span<F, 2, 4, NR, NT, NP, VEC>(a, grid, s);
    default: return launch_span<F, 4, 4, NR, NT, NP, VEC>(a, grid, s);
  }
}

}  // namespace rk
