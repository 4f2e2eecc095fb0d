// rk_span_dev.h -- one token's attention over spans of plain or quantised
// rows (MI355X, gfx950), included by the per-format units rk_span_*.hip.
//
// For a query row r and the tokens t of its spans
//   s_rt = (k_t . q_r + bias_r) log2(e) / sqrt(D),  o_r = sum_t 2^s_rt v_t,
//   l_r = sum_t 2^s_rt,  all under a running maximum m_r;
// a workgroup covers one chunk of one span for one unit of query rows and
// leaves (m, l, o) for each row: a record.  span_merge_kernel joins a row's records,
// or, behind tiles, the launch that attends the suffix.
//
// Units.  A unit is up to 16 query rows that read the same K and V: of the heads
// of a KV group, or, over a span that the batch shares, of all the batch's
// queries on a KV head.  Units of the same rows run on one XCD, whose L2 serves
// all but the first.  (32 rows to a unit need more registers than leave three
// workgroups on a CU: 17 to 32 queries on the same rows took 14.1 .. 56 us in
// ten shapes, two units of 16 take 13.1 .. 32 us.)
//
// A workgroup is four waves that take interleaved blocks of 32 tokens.  Rows
// come straight from memory into registers in the matrix core's layout, so a
// block costs no LDS traffic and no barrier:
//   S^T = K Q^T   v_mfma_f32_16x16x32: A = K, 16 tokens x 32 channels.  A
//                 lane's four-lane-group g holds whole 8-channel pieces, and
//                 any order of channels will do as long as Q has the same;
//   O^T += V^T P^T  A = V^T: a lane holds eight tokens of VB channels as it
//                 loads them and transposes them in registers.  P^T is the
//                 lane's own eight scores: lane (g, n) gets tokens 4g .. 4g + 3
//                 and 16 + 4g .. 16 + 4g + 3 of query n.
// Quantised rows are widened to bf16 by the conversion that applies the block's
// scale; queries then enter as one, two or three bf16 terms, in which bf16, fp16
// and fp32 are exact.  bf16 holds code 2^e exactly, but for 8-bit blocks whose
// largest value is below 2^-116: their smallest codes lie under bf16's least step.
//
// Loads run ahead of the products: the K registers are reloaded with the
// wave's next block as soon as the scores are formed, the V registers as soon
// as V^T is.  (Two blocks ahead: 47.9 us where one takes 45.4, 4-bit rows; 452
// and 435, 8-bit ones.)  All offsets of a lane are fixed; a block moves the
// wave-uniform base alone.  The last block of a span starts 32 rows before its
// end, its rows of the block before it left out.
//
// What bounds it.  8-bit rows of one head each, 2.9 GB: 435 us, 6.7 TB/s, HBM.
// 4-bit rows of seven heads, 186 MB: 42 us, 4.4 TB/s; per 32 rows a wave issues
// about 90 vector and 22 matrix instructions, which 12 waves on a CU fit into
// 60 % of the time; the rest waits for rows.  One request over 13 MB: 10 us, of
// them 4 to launch, rotate the queries and fetch the first rows.
#pragma once

#include <math.h>

#include "rk_common.h"
#include "rk_span.h"

namespace rk {

// ------------------------------------------------------------ row formats
// kw: 32-bit words of eight channels.
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

// The scale of byte r of w as the conversions take it: they read the exponent
// field of the operand alone (255 makes NaN), so what else the shift leaves
// does not matter.
__device__ __forceinline__ float mx_scale(uint32_t w, int r) {
  return __builtin_bit_cast(float, r < 3 ? w << (23 - 8 * r) : w >> 1);
}

// Eight channels as a matrix operand.
template <class F>
__device__ __forceinline__ uint4 widen8(const uint32_t* w, float sc) {
  if constexpr (F::kMx)
    return make_uint4(F::template pair<0>(w, sc), F::template pair<1>(w, sc), F::template pair<2>(w, sc),
                      F::template pair<3>(w, sc));
  else
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A block of 32 tokens as one wave holds it.  k[tt]: the lane's 8 KB channels
// of token 16 tt + n; v[r]: its VB channels of token token_of(g, r).  (A tile's
// 16 rows are neighbours: the 16 lanes that load one piece of them touch the
// fewest cache lines.)
__device__ __forceinline__ int token_of(int g, int r) { return 16 * (r >> 2) + 4 * g + (r & 3); }
template <class F, int KB, int VB>
struct Block {
  static constexpr int kvw = VB == 8 ? F::kw : (F::kw + 1) / 2;
  uint32_t k[2][KB * F::kw];
  uint32_t v[8][kvw];
  uint32_t ks[2];
  uint2 vs;
};

// A unit's rows of one tensor as a buffer: a load is descriptor + scalar
// offset of the block + fixed 32-bit offset of the lane (an address needs two
// registers and a 64-bit vector addition per load).  The hardware would check
// the lane's offset alone, so the kernels clamp rows and columns themselves.
typedef __amdgpu_buffer_rsrc_t Rsrc;
__device__ __forceinline__ Rsrc make_rsrc(const void* p) {
  const uint64_t v = (uint64_t)p;
  const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32;
  return __builtin_amdgcn_make_buffer_rsrc((void*)u, 0, -1, 0x00027000);  // 2^32 - 1 bytes
}
// AUX 2: non-temporal, for rows that one instruction reads whole lines of (447
// against 451 us over 2.9 GB of 8-bit rows; the half lines of 4-bit rows came from
// memory twice, so those go through the caches).  The rule is the format's alone.
// Where several row blocks read the same rows it goes either way; us, with and
// without: bf16, one block, 8 heads behind 32768 rows 29.8 and 35.5; two blocks 38.1
// and 40.7, of 4 heads behind 16384 17.9 and 16.6; 8-bit, four blocks, 8 heads behind
// 65536 71.8 and 68.5.
template <int N, int AUX = 0>
__device__ __forceinline__ void load_words(Rsrc r, uint32_t off, uint32_t base, uint32_t* w) {
  if constexpr (N == 4) {
    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, base, AUX));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, off, base, AUX));
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, base, AUX);
  }
}

// A unit's rows of one span, and a lane's byte offsets in a block.
template <int KB>
struct SpanLane {
  Rsrc k, v, ksc;
  const uint8_t* vsc;
  uint32_t ko[2], kc[KB], so[2], vo[8], vso;
};

template <class F, int KB, int VB>
__device__ __forceinline__ void lane_offsets(const Span& sp, int D, int g, int n, SpanLane<KB>& x) {
  const uint32_t last = (uint32_t)sp.S - 1;  // a span of less than 32 rows repeats its last
  const int cv = n * VB < D ? n * VB : 0;    // lanes past the head's channels: any will do
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    const uint32_t t = min((uint32_t)(16 * tt + n), last);
    if constexpr (F::kMx) {
      // eight KB channels in one piece; past the row's width the first ones
      // stand in (the query is zero there)
      const uint32_t c = 8 * KB * g < sp.width ? 8 * KB * g : 0;
      x.ko[tt] = t * sp.k_ss + (F::kw == 2 ? c : c >> 1);
      x.so[tt] = (c >> 5) * sp.ksc_sn + t;
    } else {
      x.ko[tt] = 2 * t * sp.k_ss;
    }
  }
  if constexpr (!F::kMx) {
#pragma unroll
    for (int j = 0; j < KB; ++j) x.kc[j] = 2 * (32 * j + 8 * g < sp.width ? 32 * j + 8 * g : 0);
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const uint32_t t = min((uint32_t)token_of(g, r), last);
    if constexpr (F::kMx)
      x.vo[r] = t * sp.v_ss + (F::kw == 2 ? cv : cv >> 1);
    else
      x.vo[r] = 2 * (t * sp.v_ss + (uint32_t)cv);
  }
  if constexpr (F::kMx) x.vso = (cv >> 5) * sp.vsc_sn + 4 * g;
}

// First row of a block: the span's last block ends with the span.
__device__ __forceinline__ int block_row(const Span& sp, int blk) {
  return min(blk * kSpanBlk, max(sp.S - kSpanBlk, 0));
}

template <class F, int KB, int VB, bool VEC, int AUX>
__device__ __forceinline__ void load_k(const Span& sp, const SpanLane<KB>& hd, int blk, int g, Block<F, KB, VB>& x) {
  const uint32_t t0 = block_row(sp, blk), base = t0 * sp.k_ss * (F::kMx ? 1 : 2);
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    if constexpr (F::kMx) {
      constexpr int kAll = KB * F::kw;
      if constexpr (kAll == 8) {
        load_words<4>(hd.k, hd.ko[tt], base, x.k[tt]);
        load_words<4>(hd.k, hd.ko[tt] + 16, base, x.k[tt] + 4);
      } else {
        load_words<kAll, KB == 1 ? AUX : 0>(hd.k, hd.ko[tt], base, x.k[tt]);
      }
      x.ks[tt] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(hd.ksc, hd.so[tt], t0, 0);
    } else if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < KB; ++j) load_words<4>(hd.k, hd.ko[tt] + hd.kc[j], base, x.k[tt] + 4 * j);
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
              v |= (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                       hd.k, hd.ko[tt] + 2 * (uint32_t)(c + 2 * w + e) * sp.k_sd, base, 0)
                   << (16 * e);
          x.k[tt][4 * j + w] = v;
        }
      }
    }
  }
}

template <class F, int KB, int VB, bool VEC, int AUX>
__device__ __forceinline__ void load_v(const Span& sp, const SpanLane<KB>& hd, int D, int blk, int n,
                                       Block<F, KB, VB>& x) {
  const uint32_t t0 = block_row(sp, blk), base = t0 * sp.v_ss * (F::kMx ? 1 : 2);
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    if constexpr (F::kMx) {
      if constexpr (VB == 8)
        load_words<F::kw, AUX>(hd.v, hd.vo[r], base, x.v[r]);
      else if constexpr (F::kw == 2)
        load_words<1, AUX>(hd.v, hd.vo[r], base, x.v[r]);
      else
        x.v[r][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(hd.v, hd.vo[r], base, 0);
    } else if constexpr (VEC) {
      load_words<VB / 2, AUX>(hd.v, hd.vo[r], base, x.v[r]);
    } else {
      const int cv = n * VB < D ? n * VB : 0;
#pragma unroll
      for (int w = 0; w < VB / 2; ++w) {
        uint32_t v = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (cv + 2 * w + e < D)
            v |= (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                     hd.v, hd.vo[r] + 2 * ((uint32_t)(cv + 2 * w + e) * sp.v_sd - (uint32_t)cv), base, 0)
                 << (16 * e);
        x.v[r][w] = v;
      }
    }
  }
  // eight tokens' scales of the lane's block column, at any byte address
  if constexpr (F::kMx) {
    __builtin_memcpy(&x.vs.x, hd.vsc + t0 + hd.vso, 4);
    __builtin_memcpy(&x.vs.y, hd.vsc + t0 + hd.vso + 16, 4);
  }
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

// The running maximum is raised (and the sums rescaled) only when a score
// passes it by kSlack, in log2 units: a probability is then at most 2^kSlack,
// and most blocks need no exchange between lanes.  The sums are fp32, which
// scales by powers of two without loss: the slack costs no accuracy.  fp16 probabilities are
// formed as 2^kLift p (at most 2^15): those below 2^-24, not 2^-14, fall into
// fp16's subnormals.  A workgroup's record is free of both.
template <class TT>
constexpr float kLift = TT::kRk == 0 ? 10.f : 0.f;
template <class TT>
constexpr float kSlack = TT::kRk == 0 ? 5.f : 8.f;

// The running state of one wave's 16 query rows, a row a lane (n).  m: the
// maximum that the sums are relative to (0 until the row's first score above
// -infinity); top: the lane's largest score so far, relative to m and lifted.
// l: the sum of the probabilities, formed with the others as the product of P
// with ones: every register of it is the sum.
template <int VB>
struct State {
  float m, top;
  f32x4 l, acc[VB];
  __device__ __forceinline__ void clear() {
    m = 0.f;
    top = -INFINITY;
    l = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < VB; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
};
// One instruction: fmaxf quiets each operand with another.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// The largest of a row's four lanes.
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, shfl_xor(x, 16));
  return fmaxf(x, shfl_xor(x, 32));
}
template <class TT>
__device__ __forceinline__ uint4 ones() {
  const uint32_t w = TT::kRk == F16::kRk ? 0x3c003c00u : 0x3f803f80u;
  return make_uint4(w, w, w, w);
}

// Scores to sums for one block of 32 tokens: softmax of s (raw products; off:
// the addend of a score, moved with the maximum) and O^T += V^T P^T.  on: which
// of the lane's eight tokens count, unless the block is whole.  turn(w, lo, hi)
// gives V^T of channel slots 2 w and 2 w + 1: AHEAD, all of them before the
// softmax (reads of LDS, which it hides), or each as it is needed.
template <class TT, int VB, int NP, bool AHEAD, class Turn>
__device__ __forceinline__ void weigh_block(const f32x4 (&s)[2], float scale, float& off, bool whole, uint32_t on,
                                            State<VB>& st, const Turn& turn) {
  uint4 av[AHEAD ? VB : 1];
  if constexpr (AHEAD) {
#pragma unroll
    for (int w = 0; w < VB / 2; ++w) turn(w, av[2 * w], av[2 * w + 1]);
  }
  float sc[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) sc[r] = fmaf(s[r >> 2][r & 3], scale, off);
  if (!whole) {
#pragma unroll
    for (int r = 0; r < 8; ++r) sc[r] = (on >> r) & 1u ? sc[r] : -INFINITY;
  }
  float mx = max3(sc[0], sc[1], sc[2]);
  mx = max3(mx, sc[3], sc[4]);
  mx = max3(mx, sc[5], sc[6]);
  mx = max3(mx, sc[7], sc[7]);
  // (a lane whose first score this is asks as well)
  const bool raise = mx > (st.top > -INFINITY ? kSlack<TT> + kLift<TT> : -INFINITY);
  const float was = st.top;
  st.top = max3(st.top, mx, mx);
  if (__any(raise)) {
    mx = row_max(mx);
    // how far the maximum rises; the row's first scores set it
    float up = mx - kLift<TT>;
    if (row_max(was) > -INFINITY) up = fmaxf(up, 0.f);
    if (!(up > -INFINITY)) up = 0.f;
    // (first scores far below zero: the sums are zero, and 2^-up is infinite)
    const float alpha = fast_exp2(-fmaxf(up, 0.f));
#pragma unroll
    for (int j = 0; j < VB; ++j) st.acc[j] *= alpha;
    st.l *= alpha;
    st.m += up;
    st.top -= up;
    off -= up;
#pragma unroll
    for (int r = 0; r < 8; ++r) sc[r] -= up;
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) sc[r] = fast_exp2(sc[r]);
  uint4 p[NP];
  terms8<TT, NP>(sc, p);
#pragma unroll
  for (int t = 0; t < NP; ++t) st.l = TT::mfma(ones<TT>(), p[t], st.l);
  if constexpr (AHEAD) {
#pragma unroll
    for (int t = 0; t < NP; ++t)
#pragma unroll
      for (int j = 0; j < VB; ++j) st.acc[j] = TT::mfma(av[j], p[t], st.acc[j]);
  } else {
#pragma unroll
    for (int w = 0; w < VB / 2; ++w) {
      uint4 lo, hi;
      __builtin_amdgcn_sched_barrier(0);  // one pair's registers at a time
      turn(w, lo, hi);
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        st.acc[2 * w] = TT::mfma(lo, p[t], st.acc[2 * w]);
        st.acc[2 * w + 1] = TT::mfma(hi, p[t], st.acc[2 * w + 1]);
      }
    }
  }
}

// One chunk of one span: adds the wave's blocks to `st`.  MASK: a mask of
// neighbouring bytes over at least a block, a lane's eight asked for ahead of the
// block's scores.  (8 requests of 64 heads to 8000 masked tokens: 56.5 us, 68 with a
// load and a wait per token, as other masks have; in kernels that calls without a
// mask share, the registers spill and those take 3 to 30 % longer.)  pre(): stages the
// unit's queries in LDS, sq [term][row][stride] 16-bit in the lane's channel
// order, while the first blocks are on their way; it leaves the rows' biases in sbias
// and, of fp16 terms, their largest |q R| in stop (null: none).
template <class F, int KB, int VB, int NT, int NP, bool VEC, bool MASK, class Pre>
__device__ __forceinline__ void run_span(const SpanArgs& a, const Span& sp, SpanLane<KB>& hd, int b, int chunk,
                                         int wave, int lane, const uint16_t* sq, int qstride, const float* sbias,
                                         const uint32_t* stop, State<VB>& st, const Pre& pre) {
  using TT = typename F::TT;
  const int g = lane >> 4, n = lane & 15;
  int lim = min(chunk * sp.chunk + sp.chunk, sp.S);
  if (sp.len) lim = min(lim, max(sp.len[b], 0));
  lim = __builtin_amdgcn_readfirstlane(lim);  // (a loaded length sits in a vector register)
  const int blk0 = chunk * sp.chunk / kSpanBlk + wave, nblk = (lim + kSpanBlk - 1) / kSpanBlk;
  const int nw = nblk > blk0 ? (nblk - blk0 - 1) / kSpanWaves + 1 : 0;
  // past the wave's last block the loads ahead take that block again
  auto blk_of = [&](int i) { return blk0 + kSpanWaves * min(i, max(nw - 1, 0)); };
  lane_offsets<F, KB, VB>(sp, a.D, g, n, hd);
  // rows of whole lines: 16 lanes' Value channels, four rows of 32 Key channels
  constexpr int kAux = Block<F, KB, VB>::kvw * 64 >= 128 ? 2 : 0;
  Block<F, KB, VB> x;
  load_k<F, KB, VB, VEC, kAux>(sp, hd, blk_of(0), g, x);
  load_v<F, KB, VB, VEC, kAux>(sp, hd, a.D, blk_of(0), n, x);
  pre();
  // queries held in registers where that leaves room for the blocks
  constexpr bool kRegQ = NT * KB <= (F::kMx ? 4 : 8);
  uint4 qreg[kRegQ ? NT : 1][kRegQ ? KB : 1];
  auto qload = [&](int t, int j) {
    const int c = F::kMx ? 8 * KB * g + 8 * j : 32 * j + 8 * g;
    return *(const uint4*)(sq + (t * 16 + n) * qstride + c);
  };
  if constexpr (kRegQ) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < KB; ++j) qreg[t][j] = qload(t, j);
  }
  // a score is one fused multiply-add: the bias, the maximum and the lift in
  // its addend
  float off = (sbias ? sbias[n] * a.scale_log2 : 0.f) + kLift<TT>;
  float scale = a.scale_log2;
  if constexpr (TT::kRk == F16::kRk)
    if (stop) scale = ldexpf(scale, split_shift(__builtin_bit_cast(float, stop[n])));

  auto compute = [&](int blk, int next) {
    uint2 mask;
    if constexpr (MASK) {
      const uint8_t* p = sp.mask + b * sp.m_sb + block_row(sp, blk) + 4 * g;
      __builtin_memcpy(&mask.x, p, 4);
      __builtin_memcpy(&mask.y, p + 16, 4);
    }
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int j = 0; j < KB; ++j)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        uint4 kop = widen8<F>(x.k[tt] + j * F::kw, mx_scale(x.ks[tt], 0));
        // plain rows narrower than KB blocks: no value of another channel
        // meets the query's zero (an infinity would make NaN)
        if constexpr (!F::kMx && VEC)
          if (sp.width < 32 * KB && 32 * j + 8 * g >= sp.width) kop = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (kRegQ)
            s[tt] = TT::mfma(kop, qreg[t][j], s[tt]);
          else
            s[tt] = TT::mfma(kop, qload(t, j), s[tt]);
        }
      }
    load_k<F, KB, VB, VEC, kAux>(sp, hd, next, g, x);
    // which of the lane's eight tokens count
    const int t0 = block_row(sp, blk);
    uint32_t on = 0xffu;
    const bool whole = (blk + 1) * kSpanBlk <= lim && !sp.mask;
    if (!whole) {
      on = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int t = t0 + token_of(g, r);
        bool ok = t >= blk * kSpanBlk && t < lim;
        if constexpr (MASK)
          ok = ok && ((r < 4 ? mask.x : mask.y) >> (8 * (r & 3)) & 0xffu) != 0;
        else if (sp.mask && ok)
          ok = sp.mask[b * sp.m_sb + t * sp.m_ss] != 0;
        on |= (uint32_t)ok << r;
        // a row that does not count holds anything: 0 x NaN must not reach the
        // sum.  (Here, under the branch: as selects at V^T they would run in
        // every block, 64 of 233 vector instructions.)
        if constexpr (F::kMx) {
          uint32_t& vs = r < 4 ? x.vs.x : x.vs.y;
          vs = ok ? vs : vs & ~(0xffu << (8 * (r & 3)));
        }
#pragma unroll
        for (int w = 0; w < Block<F, KB, VB>::kvw; ++w) x.v[r][w] = ok ? x.v[r][w] : 0u;
      }
    }
    // V^T of channel slots 2 w and 2 w + 1: eight tokens of each
    auto turn = [&](int w, uint4& lo, uint4& hi) {
      uint32_t y[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if constexpr (F::kMx) {
          const float sc = mx_scale(r < 4 ? x.vs.x : x.vs.y, r & 3);
          y[r] = w == 0   ? F::template pair<0>(x.v[r], sc)
                 : w == 1 ? F::template pair<1>(x.v[r], sc)
                 : w == 2 ? F::template pair<2>(x.v[r], sc)
                          : F::template pair<3>(x.v[r], sc);
        } else {
          y[r] = x.v[r][w];
        }
      }
      lo = make_uint4(pack_lo(y[0], y[1]), pack_lo(y[2], y[3]), pack_lo(y[4], y[5]), pack_lo(y[6], y[7]));
      hi = make_uint4(pack_hi(y[0], y[1]), pack_hi(y[2], y[3]), pack_hi(y[4], y[5]), pack_hi(y[6], y[7]));
    };
    weigh_block<TT, VB, NP, false>(s, scale, off, whole, on, st, turn);
    load_v<F, KB, VB, VEC, kAux>(sp, hd, a.D, next, n, x);
  };

  for (int i = 0; i < nw; ++i) compute(blk_of(i), blk_of(i + 1));
}

// Query row R of a unit: its batch row and head.
struct RowOf {
  int b, h;
};
__device__ __forceinline__ RowOf row_of(const SpanArgs& a, bool shared, int b, int kv, int R) {
  RowOf o;
  o.b = shared ? R / a.G : b;
  o.h = kv * a.G + (shared ? R - o.b * a.G : R);
  return o;
}

// A unit's queries: thread i holds the i-th eight channels of every 256 of
// them (16 to a row), as they are in memory (the host sees to whole, 16-byte
// aligned pieces).  NW: 32-bit words of eight channels.
template <int NR, int NW>
struct Queries {
  uint32_t w[NR][NW];
};

template <int NR, int NW>
__device__ __forceinline__ void load_queries(const SpanArgs& a, bool shared, int b, int kv, int R0, int rows, int tid,
                                             Queries<NR, NW>& x) {
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int c = 8 * (tid & 15), r = 16 * i + (tid >> 4);
#pragma unroll
    for (int e = 0; e < NW; ++e) x.w[i][e] = 0u;
    if (r < rows && c < a.D) {
      const RowOf o = row_of(a, shared, b, kv, R0 + r);
      const char* p = (const char*)a.q + (NW / 2) * (o.b * a.q_sb + o.h * a.q_sh + c);
#pragma unroll
      for (int e = 0; e < NW; e += 4) {
        const u32x4 v = *(const u32x4*)(p + 4 * e);
        x.w[i][e] = v.x; x.w[i][e + 1] = v.y; x.w[i][e + 2] = v.z; x.w[i][e + 3] = v.w;
      }
    }
  }
}

// Eight channels of a held row as fp32.
template <int NR, int NW>
__device__ __forceinline__ void query8(const Queries<NR, NW>& x, int i, bool f16, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (NW == 8) {
      v[e] = __builtin_bit_cast(float, x.w[i][e]);
    } else {
      const uint16_t h = (uint16_t)(x.w[i][e >> 1] >> (16 * (e & 1)));
      v[e] = f16 ? F16::to_f32(h) : BF16::to_f32(h);
    }
  }
}

// ... and their NT terms of TT in LDS, [term][row][stride], zeros past the
// head's channels and the unit's rows; channels up to kW.
template <class TT, int NT, int NR, int NW, int kW>
__device__ __forceinline__ void stage_queries(int tid, const Queries<NR, NW>& x, bool f16, uint16_t* dst, int stride) {
  const int c = 8 * (tid & 15);
  if (c >= kW) return;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    uint4 t[NT];
    if constexpr (NT == 1) {
      t[0] = make_uint4(x.w[i][0], x.w[i][1], x.w[i][2], x.w[i][3]);
    } else {
      float v[8];
      query8(x, i, f16, v);
      terms8<TT, NT>(v, t);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) *(uint4*)(dst + (j * 16 * NR + 16 * i + (tid >> 4)) * stride + c) = t[j];
  }
}

// The rotation of a unit's queries where q, R_partial and delta_mu share one
// 16-bit type and lie in whole 16-byte pieces; other calls find q R and the
// biases formed ahead (span_queries_kernel).
//
// Each thread's pieces of R, and of delta_mu.
template <int KV>
struct Rotation {
  u32x4 r[2 * KV], mu;
};

template <int KV>
__device__ __forceinline__ void load_rotation(const SpanArgs& a, int rb, int kv, int tid, Rotation<KV>& x) {
  const uint16_t* R = (const uint16_t*)a.R + rb * a.R_sb + kv * a.R_sh;
#pragma unroll
  for (int i = 0; i < 2 * KV; ++i) {
    const int id = i * kSpanThreads + tid, d = id / (4 * KV), c = 8 * (id % (4 * KV));
    x.r[i] = (u32x4){0u, 0u, 0u, 0u};
    if (d < a.D && c < a.Dk) x.r[i] = *(const u32x4*)(R + d * a.R_sd + c);
  }
  x.mu = (u32x4){0u, 0u, 0u, 0u};
  if (a.dm && 8 * tid < a.D) x.mu = *(const u32x4*)((const uint16_t*)a.dm + rb * a.dm_sb + kv * a.dm_sh + 8 * tid);
}

// Where piece p of row r lies for a transposing read, which takes 32
// neighbouring bytes of 16 rows: rows of P pieces (4, 8, 16), eight rows' 32
// bytes fill the banks once.
template <int P>
__device__ __forceinline__ int swizzle_v(int p, int r) {
  return p ^ (2 * ((r / (16 / P)) & (P / 2 - 1)));
}

// Columns 16 j .. 16 j + 15 of the rows r0 + 4 g .. + 3 and r0 + 16 + 4 g .. + 3
// of a matrix in LDS (rows of P swizzled pieces), a column a lane: lane 4 t + q of
// 16 names row t, columns 4 q .. 4 q + 3, and receives its column of all four.
template <int P>
__device__ __forceinline__ uint4 read_columns(const void* m, int r0, int j, int g, int n) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4* lptr;
  uint2 x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + 16 * i + 4 * g + (n >> 2), p = 2 * j + ((n >> 1) & 1);
    const char* at = (const char*)m + 16 * (r * P + swizzle_v<P>(p, r)) + 8 * (n & 1);
    x[i] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)at));
  }
  return make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
}

template <int KV>
__device__ __forceinline__ void stage_rotation(int tid, const Rotation<KV>& x, uint4* r, uint4* mu) {
#pragma unroll
  for (int i = 0; i < 2 * KV; ++i) {
    const int id = i * kSpanThreads + tid, d = id / (4 * KV), p = id % (4 * KV);
    r[d * (4 * KV) + swizzle_v<4 * KV>(p, d)] = make_uint4(x.r[i].x, x.r[i].y, x.r[i].z, x.r[i].w);
  }
  if (tid < 16) mu[tid] = make_uint4(x.mu.x, x.mu.y, x.mu.z, x.mu.w);
}

// raw: the queries as they are, [row][136]; r, mu: the staged rotation.  q R is
// left as NTV terms of TT in `dst`, q . delta_mu in `bias`, behind a barrier.  A wave
// takes tiles of 16 columns; one more has delta_mu in every column.  (Channel order
// within 32: as read_columns gives them.)  fp16 terms: `top`, zero before, gets the
// largest |q R| of the rows that pass kSplitTop; if one does, all form their terms
// again, those rows scaled.
template <class TT, int NTV, int NR, int KV>
__device__ __forceinline__ void rotate_queries(const SpanArgs& a, int wave, int lane, bool f16, const uint16_t* raw,
                                               const uint4* r, const uint4* mu, uint16_t* dst, int stride,
                                               float* bias, uint32_t* top) {
  constexpr int kRows = 16 * NR;
  constexpr bool kScaled = TT::kRk == F16::kRk;
  const int g = lane >> 4, n = lane & 15;
  for (bool again = false;; again = true) {
    for (int ct = wave; ct <= 2 * KV; ct += kSpanWaves) {
      f32x4 o[NR];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) o[nr] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint4 m;
        if (ct < 2 * KV) {
          m = read_columns<4 * KV>(r, 32 * ks, ct, g, n);
        } else {
          const uint2 lo = ((const uint2*)mu)[8 * ks + g], hi = ((const uint2*)mu)[8 * ks + 4 + g];
          m = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          const uint2* p = (const uint2*)(raw + (16 * nr + n) * 136 + 32 * ks);
          const uint4 q = make_uint4(p[g].x, p[g].y, p[4 + g].x, p[4 + g].y);
          o[nr] = f16 ? F16::mfma(q, m, o[nr]) : BF16::mfma(q, m, o[nr]);
        }
      }
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = o[nr][i];
          const int row = 16 * nr + 4 * g + i;
          if (ct == 2 * KV) {
            if (n == 0) bias[row] = v;
          } else {
            if constexpr (kScaled) {
              if (again)
                v = ldexpf(v, -split_shift(__builtin_bit_cast(float, top[row])));
              else if (fabsf(v) >= kSplitTop)
                atomicMax(top + row, __builtin_bit_cast(uint32_t, fabsf(v)));
            }
#pragma unroll
            for (int k = 0; k < NTV; ++k) {
              const uint16_t h = TT::from_f32(v);
              dst[(k * kRows + row) * stride + ct * 16 + n] = h;
              v -= TT::to_f32(h);
            }
          }
        }
    }
    __syncthreads();
    // (the same in every wave: nothing writes `top` any more)
    if (!kScaled || again || !__any(top[lane & (kRows - 1)] != 0u)) break;
  }
}

// Four output channels of a row, in the output's dtype.
__device__ __forceinline__ void store_out4(const SpanArgs& a, int64_t b, int64_t h, int c, f32x4 v) {
  const int64_t off = b * a.o_sb + h * a.o_sh + c * a.o_sd;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (c + e >= a.D) break;
    const int64_t at = off + e * a.o_sd;
    if (a.o_dtype == F32::kRk)
      ((float*)a.out)[at] = v[e];
    else
      ((uint16_t*)a.out)[at] = a.o_dtype == F16::kRk ? F16::from_f32(v[e]) : BF16::from_f32(v[e]);
  }
}

// Four channels of a row's suffix sums (M, L, v) joined with the records of the
// spans before it, eight records' loads in flight, and written out.
template <int DV>
__device__ __forceinline__ void join_records(const SpanArgs& a, const RowOf& o, int c, float M, float L, f32x4 v) {
  constexpr int NB = 8;
  const int64_t at = ((int64_t)o.b * a.Hq + o.h) * a.np;
  const float2* ml = (const float2*)a.ml + at;
  const float* acc = a.acc + at * DV + c;
  for (int p = 0; p < a.np; p += NB) {
    float2 r[NB];
    f32x4 x[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int q = min(p + i, a.np - 1);  // past the last: it again, with weight 0
      r[i] = ml[q];
      x[i] = *(const f32x4*)(acc + (int64_t)q * DV);
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < NB; ++i) top = fmaxf(top, r[i].x);
    const float f = fast_exp2(M - top);
    M = top;
    L *= f;
    v *= f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const float w = p + i < a.np ? fast_exp2(r[i].x - M) : 0.f;
      L = fmaf(r[i].y, w, L);
      v += x[i] * w;
    }
  }
  store_out4(a, o.b, o.h, c, v / (L + kDenomEps));
}

// JOIN: the launch behind tile_kernel's, over the suffix rows of a shared call
// (one workgroup per unit).  It joins the other spans' records to its sums and
// writes the output.
//
// Registers: 128 a lane for quantised rows (four workgroups on a CU, of which the
// plan fills three and the fourth takes a late one), 168 for plain ones, whose
// blocks are twice as wide, 256 for element loads (VEC false), which keep an
// address per element.
template <class F, int KV, int KF, int NT, int NP, bool VEC, bool MASK, bool JOIN>
__global__ void __launch_bounds__(kSpanThreads, VEC ? (F::kMx ? 4 : 3) : 2) span_kernel(const SpanArgs a) {
  using TT = typename F::TT;
  constexpr int VB = KF == 2 ? 4 : 8;
  constexpr int DV = 16 * VB;
  constexpr int NTV = NT < 2 ? 2 : NT;  // terms of a rotated query
  constexpr int NW = NT == 3 ? 8 : 4;   // words of eight channels of a query
  constexpr int kRows = 16;
  constexpr int kWide = 32 * (KV > KF ? KV : KF) + 8;  // +8: rows start in other banks
  constexpr int kQ = kRows * kWide * (KV > 0 ? NTV : NT);
  constexpr int kRaw = KV > 0 && NT < 3 ? kRows * 136 + 128 * 32 * KV + 128 : 0;
  constexpr int kAccRow = DV + 4;       // floats; +4: rows start in other banks
  constexpr int kAcc = kSpanWaves * kRows * kAccRow;
  __shared__ __attribute__((aligned(16))) char s_mem[(kQ + kRaw) * 2 > kAcc * 4 ? (kQ + kRaw) * 2 : kAcc * 4];
  __shared__ float s_bias[kRows];
  constexpr bool kScaled = KV > 0 && TT::kRk == F16::kRk;
  __shared__ uint32_t s_qtop[kScaled ? kRows : 1];
  __shared__ float s_m[kSpanWaves][kRows], s_top[kSpanWaves][kRows], s_l[kSpanWaves][kRows];
  uint16_t* s_q = (uint16_t*)s_mem;
  uint16_t* s_raw = s_q + kQ;
  float* s_acc = (float*)s_mem;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int id = (int)blockIdx.x;
  const int k = JOIN || id >= a.first[kTail] ? kTail : id >= a.first[kFull] ? kFull : kRotated;
  const Span sp = a.span[k];  // (copied whole: few, wide scalar loads)
  const int rel = JOIN ? id : id - a.first[k];
  // Workgroups go to the 8 XCDs, each with an L2 of its own, in turn: the row
  // blocks that read the same rows are 8 ids apart, on one XCD.  The last of the
  // ids may have none.
  // (Quotients are formed on the vector unit: back to scalar registers, so that
  // everything derived from them stays there.)
  const bool shared = a.shared && k != kTail;
  const int blocks = a.blocks[k], heads = a.heads[k];
  const int q8 = __builtin_amdgcn_readfirstlane((rel >> 3) / blocks);
  const int t = 8 * q8 + (rel & 7), R0 = ((rel >> 3) - q8 * blocks) * kRows;
  const int x = __builtin_amdgcn_readfirstlane(t / heads), ukv = t - x * heads;
  if (x >= sp.wgs) return;
  const int b = shared ? 0 : __builtin_amdgcn_readfirstlane(ukv / a.H), kv = shared ? ukv : ukv - b * a.H;
  const int rows = min((shared ? a.B * a.G : a.G) - R0, kRows);

  State<VB> st;
  st.clear();

  auto head = [&](auto& hd) {
    constexpr int kEl = F::kMx ? 1 : 2;
    hd.k = make_rsrc((const char*)sp.k + kEl * (b * sp.k_sb + kv * sp.k_sh));
    hd.v = make_rsrc((const char*)sp.v + kEl * (b * sp.v_sb + kv * sp.v_sh));
    if constexpr (F::kMx) {
      hd.ksc = make_rsrc(sp.ksc + b * sp.ksc_sb + kv * sp.ksc_sh);
      hd.vsc = sp.vsc + b * sp.vsc_sb + kv * sp.vsc_sh;
    }
  };
  // The small loads first: loads return in order, and nothing below then waits
  // for the first K and V block.
  const bool f16 = F::kMx ? a.q_dtype == F16::kRk : TT::kRk == F16::kRk;
  Queries<1, NW> qw;
  bool done = false;
  if constexpr (KV > 0) {
    if (k == kRotated) {
      SpanLane<KV> hd;
      head(hd);
      const bool here = NT < 3 && !a.qr;
      Rotation<KV> rot;
      if (here) {
        load_queries<1, NW>(a, shared, b, kv, R0, rows, tid, qw);
        load_rotation<KV>(a, shared ? 0 : b, kv, tid, rot);
      }
      auto pre = [&]() {
        if (here) {
          if constexpr (NT < 3) {
            uint4* s_r = (uint4*)(s_raw + kRows * 136);
            uint4* s_mu = s_r + 128 * 4 * KV;
            stage_queries<TT, 1, 1, NW, 128>(tid, qw, f16, s_raw, 136);
            stage_rotation<KV>(tid, rot, s_r, s_mu);
            if constexpr (kScaled)
              if (tid < kRows) s_qtop[tid] = 0u;
            __syncthreads();
            rotate_queries<TT, NTV, 1, KV>(a, wave, lane, f16, s_raw, s_r, s_mu, s_q, kWide, s_bias, s_qtop);
          }
        } else {
          constexpr int W = 32 * KV;
          for (int i = tid; i < NTV * kRows * (W / 8); i += kSpanThreads) {
            const int c = 8 * (i % (W / 8)), r = (i / (W / 8)) % kRows, t = i / (W / 8) / kRows;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < rows) {
              const RowOf o = row_of(a, shared, b, kv, R0 + r);
              v = *(const uint4*)(a.qr + (((int64_t)o.b * a.Hq + o.h) * NTV + t) * W + c);
            }
            *(uint4*)(s_q + (t * kRows + r) * kWide + c) = v;
          }
          if (tid < kRows) {
            const RowOf o = row_of(a, shared, b, kv, R0 + min(tid, rows - 1));
            s_bias[tid] = a.bias[(int64_t)o.b * a.Hq + o.h];
            if constexpr (kScaled) s_qtop[tid] = __builtin_bit_cast(uint32_t, a.qtop[(int64_t)o.b * a.Hq + o.h]);
          }
          __syncthreads();
        }
      };
      run_span<F, KV, VB, NTV, NP, VEC, false>(a, sp, hd, b, x, wave, lane, s_q, kWide, s_bias,
                                               kScaled ? s_qtop : nullptr, st, pre);
      done = true;
    }
  }
  if (!done) {
    SpanLane<KF> hd;
    head(hd);
    load_queries<1, NW>(a, shared, b, kv, R0, rows, tid, qw);
    auto pre = [&]() {
      stage_queries<TT, NT, 1, NW, 32 * KF>(tid, qw, f16, s_q, kWide);
      __syncthreads();
    };
    run_span<F, KF, VB, NT, NP, VEC, MASK>(a, sp, hd, b, x, wave, lane, s_q, kWide, nullptr, nullptr, st, pre);
  }

  // The row's true maximum; a row without tokens has the least one.
  float top = row_max(st.top);
  const bool seen = top > -INFINITY;
  top = seen ? top + st.m - kLift<TT> : kNegInit;
  const float m = seen ? st.m : kNegInit;
  // join the four waves: the common maximum, every wave's sums under it through
  // LDS, then a thread adds four channels of a row
  if (g == 0) {
    s_m[wave][n] = m;
    s_top[wave][n] = top;
    s_l[wave][n] = st.l[0];
  }
  __syncthreads();  // (also: no wave reads queries any more)
  if (n < rows) {
    const float M = fmaxf(fmaxf(s_top[0][n], s_top[1][n]), fmaxf(s_top[2][n], s_top[3][n]));
    const float f = fast_exp2(m - M - kLift<TT>);
    float* dst = s_acc + (wave * kRows + n) * kAccRow + 4 * g * VB;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VB; j += 4)
        *(f32x4*)(dst + i * VB + j) = (f32x4){st.acc[j][i] * f, st.acc[j + 1][i] * f, st.acc[j + 2][i] * f,
                                              st.acc[j + 3][i] * f};
  }
  __syncthreads();
  const int rec = sp.np0 + x;
  for (int i = tid; i < rows * (DV / 4); i += kSpanThreads) {
    const int r = i / (DV / 4), c = 4 * (i % (DV / 4));
    f32x4 v = *(const f32x4*)(s_acc + r * kAccRow + c);
#pragma unroll
    for (int w = 1; w < kSpanWaves; ++w) v += *(const f32x4*)(s_acc + (w * kRows + r) * kAccRow + c);
    const RowOf o = row_of(a, shared, b, kv, R0 + r);
    const int64_t at = ((int64_t)o.b * a.Hq + o.h) * a.np + rec;
    if (JOIN || c == 0) {
      const float M = fmaxf(fmaxf(s_top[0][r], s_top[1][r]), fmaxf(s_top[2][r], s_top[3][r]));
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < kSpanWaves; ++w) L += s_l[w][r] * fast_exp2(s_m[w][r] - M - kLift<TT>);
      if constexpr (JOIN)
        join_records<DV>(a, o, c, M, L, v);
      else
        *(float2*)(a.ml + 2 * at) = make_float2(M, L);
    }
    if constexpr (!JOIN) *(f32x4*)(a.acc + at * DV + c) = v;
  }
}

template <class F, int KV, int KF, int NT, int NP, bool VEC>
hipError_t launch_span(const SpanArgs& a, unsigned grid, hipStream_t s) {
  if constexpr (F::kMx) {  // (plain rows are a shared call's, which has no mask)
    const Span& sp = a.span[kFull];
    if (sp.mask && sp.m_ss == 1 && sp.S >= kSpanBlk) {
      hipLaunchKernelGGL((span_kernel<F, KV, KF, NT, NP, VEC, true, false>), dim3(grid), dim3(kSpanThreads), 0, s, a);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((span_kernel<F, KV, KF, NT, NP, VEC, false, false>), dim3(grid), dim3(kSpanThreads), 0, s, a);
  return hipGetLastError();
}

// The instantiation for a call's widths.
template <class F, int NT, int NP, bool VEC>
hipError_t pick_widths(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s) {
  if (kf == 2) {
    switch (kv) {
      case 0: return launch_span<F, 0, 2, NT, NP, VEC>(a, grid, s);
      case 1: return launch_span<F, 1, 2, NT, NP, VEC>(a, grid, s);
      default: return launch_span<F, 2, 2, NT, NP, VEC>(a, grid, s);
    }
  }
  switch (kv) {
    case 0: return launch_span<F, 0, 4, NT, NP, VEC>(a, grid, s);
    case 1: return launch_span<F, 1, 4, NT, NP, VEC>(a, grid, s);
    case 2: return launch_span<F, 2, 4, NT, NP, VEC>(a, grid, s);
    default: return launch_span<F, 4, 4, NT, NP, VEC>(a, grid, s);
  }
}

// The suffix rows of a shared call and the join (kf as above).
template <class F, int NT, int NP>
hipError_t pick_join(int kf, const SpanArgs& a, unsigned grid, hipStream_t s) {
  if (kf == 2)
    hipLaunchKernelGGL((span_kernel<F, 0, 2, NT, NP, true, false, true>), dim3(grid), dim3(kSpanThreads), 0, s, a);
  else
    hipLaunchKernelGGL((span_kernel<F, 0, 4, NT, NP, true, false, true>), dim3(grid), dim3(kSpanThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace rk
