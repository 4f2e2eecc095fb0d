// rk_span.hip -- host side of the attention over quantised and shared spans
// (rk_quantized_decode, rk_shared_prefix_decode of rotatek_hip.h): validation,
// the split plan and the launches, and the small kernels beside the split one
// (rk_span_dev.h, rk_tile_dev.h): queries that it does not take as they are,
// and the join of a row's partial sums.
#include <hip/hip_runtime.h>
#include <string.h>

#include <algorithm>

#include "rk_common.h"
#include "rk_host.h"
#include "rk_mx.h"
#include "rk_span.h"
#include "rotatek_hip.h"

namespace {

using rk::kFull;
using rk::kRotated;
using rk::kSpans;
using rk::kTail;
using rk::Span;
using rk::SpanArgs;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

// ---------------------------------------------------------------- kernels

// The queries of calls in other layouts and types, a row per workgroup: a
// padded copy, and q R_partial and q . delta_mu in fp32, q R stored as a sum of
// `terms` 16-bit values (two hold 16 or more bits of it, three an fp32's 24).
__global__ void __launch_bounds__(128) span_queries_kernel(const rk::QueryArgs a) {
  __shared__ float s_q[128];
  __shared__ float s_b[2], s_t[2];
  const int c = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int64_t b = row / a.Hq, h = row - b * a.Hq, kv = h / a.G, rb = a.shared ? 0 : b;
  const float q = c < a.D ? rk::load_any(a.q, b * a.q_sb + h * a.q_sh + c * a.q_sd, a.q_dtype) : 0.f;
  s_q[c] = q;
  if (a.q_out && c < a.Dp) {
    if (a.q_dtype == RK_F32)
      ((float*)a.q_out)[row * a.Dp + c] = q;
    else
      ((uint16_t*)a.q_out)[row * a.Dp + c] = a.q_dtype == RK_F16 ? rk::F16::from_f32(q) : rk::BF16::from_f32(q);
  }
  if (!a.qr) return;
  __syncthreads();
  float v = 0.f;
  if (c < a.Dk) {
    const int64_t off = rb * a.R_sb + kv * a.R_sh + c * a.R_sk;
    for (int d = 0; d < a.D; d += 32) {
      float r[32];
      rk::load_any_rows<32>(a.R, off, a.R_sd, a.r_dtype, d, a.D, r);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (d + i < a.D) v = fmaf(s_q[d + i], r[i], v);
    }
  }
  if (a.f16) {
    float top = fabsf(v);
    for (int d = 32; d; d >>= 1) top = fmaxf(top, rk::shfl_xor(top, d));
    if ((c & 63) == 0) s_t[c >> 6] = top;
    __syncthreads();
    top = fmaxf(s_t[0], s_t[1]);
    if (c == 0) a.qtop[row] = top;
    v = ldexpf(v, -rk::split_shift(top));
  }
  if (c < a.W) {
    for (int t = 0; t < a.terms; ++t) {
      const uint16_t w = a.f16 ? rk::F16::from_f32(v) : rk::BF16::from_f32(v);
      a.qr[(row * a.terms + t) * a.W + c] = w;
      v -= a.f16 ? rk::F16::to_f32(w) : rk::BF16::to_f32(w);
    }
  }
  float p = 0.f;
  if (a.dm && c < a.D) p = q * rk::load_any(a.dm, rb * a.dm_sb + kv * a.dm_sh + c * a.dm_sd, a.dm_dtype);
  for (int d = 32; d; d >>= 1) p += rk::shfl_xor(p, d);
  if ((c & 63) == 0) s_b[c >> 6] = p;
  __syncthreads();
  if (c == 0) a.bias[row] = s_b[0] + s_b[1];
}

// Joins a row's records: out = sum_p acc_p 2^(m_p - M) / (sum_p l_p 2^(m_p -
// M) + 1e-6).  W waves to a row: each has four groups of 16 lanes (DV / 16
// channels a lane), and a group folds every 4 W-th record, four records' loads
// in flight; groups are combined by lane exchange, waves through LDS.
// Bound by the latency of its rounds, 16 W records each: a call with 28 rows of
// 190 records takes 15.5 us with four waves to a row, 23.7 with one.
template <int DV, int W>
__global__ void __launch_bounds__(256) span_merge_kernel(const SpanArgs a) {
  constexpr int C = DV / 16, NB = 4, kStep = 4 * W;
  __shared__ float s_part[W][16][C + 2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, s = lane >> 4, n = lane & 15;
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + wave / W;
  if (row >= (int64_t)a.B * a.Hq) return;  // (W 4: the whole workgroup)
  const float* acc = a.acc + row * a.np * DV + n * C;
  const float2* ml = (const float2*)a.ml + row * a.np;
  float M = rk::kNegInit, L = 0.f, A[C];
#pragma unroll
  for (int e = 0; e < C; ++e) A[e] = 0.f;
  for (int p = s + 4 * (wave % W); p < a.np; p += kStep * NB) {
    float2 r[NB];
    float4 v[NB][C / 4];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int q = p + kStep * i < a.np ? p + kStep * i : p;  // past the last: a record again, with weight 0
      r[i] = ml[q];
#pragma unroll
      for (int e = 0; e < C / 4; ++e) v[i][e] = *(const float4*)(acc + (int64_t)q * DV + 4 * e);
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < NB; ++i) top = fmaxf(top, r[i].x);
    const float f = rk::fast_exp2(M - top);
    M = top;
    L *= f;
#pragma unroll
    for (int e = 0; e < C; ++e) A[e] *= f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (p + kStep * i >= a.np) break;
      const float w = rk::fast_exp2(r[i].x - M);
      L += r[i].y * w;
#pragma unroll
      for (int e = 0; e < C / 4; ++e) {
        A[4 * e] += v[i][e].x * w; A[4 * e + 1] += v[i][e].y * w;
        A[4 * e + 2] += v[i][e].z * w; A[4 * e + 3] += v[i][e].w * w;
      }
    }
  }
#pragma unroll
  for (int d = 16; d < 64; d <<= 1) {
    const float Mo = rk::shfl_xor(M, d), top = fmaxf(M, Mo);
    const float f = rk::fast_exp2(M - top), fo = rk::fast_exp2(Mo - top);
    L = L * f + rk::shfl_xor(L, d) * fo;
#pragma unroll
    for (int e = 0; e < C; ++e) A[e] = A[e] * f + rk::shfl_xor(A[e], d) * fo;
    M = top;
  }
  if constexpr (W > 1) {
    if (s == 0) {
      s_part[wave][n][C] = M;
      s_part[wave][n][C + 1] = L;
#pragma unroll
      for (int e = 0; e < C; ++e) s_part[wave][n][e] = A[e];
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float* o = s_part[w][n];
      const float top = fmaxf(M, o[C]), f = rk::fast_exp2(M - top), fo = rk::fast_exp2(o[C] - top);
      L = L * f + o[C + 1] * fo;
#pragma unroll
      for (int e = 0; e < C; ++e) A[e] = A[e] * f + o[e] * fo;
      M = top;
    }
  }
  if (s != 0) return;
  const int64_t b = row / a.Hq, h = row - b * a.Hq;
  const int64_t off = b * a.o_sb + h * a.o_sh;
  const float den = L + rk::kDenomEps;
#pragma unroll
  for (int e = 0; e < C; ++e) {
    const int c = n * C + e;
    if (c >= a.D) break;
    const float v = A[e] / den;
    const int64_t at = off + c * a.o_sd;
    if (a.o_dtype == RK_F32)
      ((float*)a.out)[at] = v;
    else
      ((uint16_t*)a.out)[at] = a.o_dtype == RK_F16 ? rk::F16::from_f32(v) : rk::BF16::from_f32(v);
  }
}

// Rotated rows without channels: what the kernels read in their place is zero.
__global__ void __launch_bounds__(256) span_zero_kernel(uint32_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0u;
}

// ------------------------------------------------------------------- host

// Rows that many queries share: from this many bytes of a token's K and V, times
// blocks of 16 queries, the waves of a workgroup take queries (tile_kernel), below
// it tokens, and the row blocks read the rows from one L2 (span_kernel).  Tiles and
// tokens behind 16384 rows, us: 64 queries of 512 bytes 31.1 and 36.4, 128 34.8 and
// 57.6; of 256 bytes 96 39.0 and 34.7, 128 39.7 and 41.1, 256 60.2 and 65.1; of 128
// bytes 192 47.5 and 39.8, 256 51.6 and 48.8.  448 of 160 bytes behind 32768: 64 and
// 73.
constexpr int64_t kTileBytes = 2048;
// Suffix rows up to this many are attended in the launch that joins the tiles'
// records, one workgroup per request and KV head, for a launch less: 64 requests
// of 4 KV heads with 2000 tokens 84 us, with a launch each 122; 48 of 2 heads,
// too few to fill the chip, 43.8 and 42.3.  (Without tiles the suffix is split
// with the other spans: 2 requests of 4 heads 11.3 us, joined 12.9.)
constexpr int64_t kJoinTokens = 4096;
// Records that one wave joins; four take more.  (A call of 32 rows of 19 records:
// 14.7 us with one wave to a row, 13.7 with four; 1024 rows of 5: equal.)
constexpr int64_t kMergeWave = 8;
// Bytes a workgroup streams at most.
constexpr int64_t kMaxShare = INT64_C(512) << 10;

// A launch has less than 2^32 threads.
constexpr int64_t kMaxGrid = INT64_C(1) << 24;

// One call as the entry points give it; pairs may be null.
struct Call {
  const rk_tensor *q, *R, *dm, *mask, *out;
  const rk_rows* k[kSpans];
  const rk_rows* v[kSpans];
  const int32_t* len[kSpans];
  int64_t groups;
  bool shared;
};

struct Plan {
  int64_t B, Hq, H, G, D, Dk;
  int format, kv, kf, terms;
  bool vec, join;  // join: the suffix rows run in the launch that joins the tiles' records
  bool tile;       // rk_tile_dev.h over the shared spans, 64 queries a workgroup
  bool copy_q, ahead;  // queries copied into whole pieces; rotated ahead of the split launch
  int64_t S[kSpans], chunk[kSpans], wgs[kSpans], units[kSpans], blocks[kSpans], np, rows;
  size_t q, qr, bias, qtop, zero, zero_bytes, acc, ml, total;
};

// Workgroup ids of a span: eight (chunk, head) pairs' row blocks at a time.  (A
// batch of none has no row blocks over shared rows.)
int64_t launched(const Plan& p, int i) {
  return p.S[i] == 0 || p.units[i] == 0 ? 0 : 8 * p.blocks[i] * cdiv(p.wgs[i] * (p.units[i] / p.blocks[i]), 8);
}

bool mx(const rk_rows* r) { return r->format != RK_ROWS_PLAIN; }

// Rows of one span: shape [N, H, S, dim], one format and, if plain, q's dtype.
int check_rows(const rk_rows* r, int format, int dtype, int64_t N, int64_t H, int64_t S, int64_t dim) {
  if (!r) return RK_ERR_NULL;
  if (r->format != format) return RK_ERR_DTYPE;
  if (mx(r)) {
    const int st = rk::check_mx(r);
    if (st) return st;
    if (r->head_dim != dim) return RK_ERR_SHAPE;
  } else {
    const int st = rk::check_desc(&r->data, 4);
    if (st) return st;
    if (r->data.dtype != dtype) return RK_ERR_DTYPE;
    if (r->data.shape[3] != dim || r->head_dim != dim) return RK_ERR_SHAPE;
    // 32-bit byte offsets inside a head
    if ((S + 64) * r->data.stride[2] + dim * r->data.stride[3] >= (INT64_C(1) << 31)) return RK_ERR_STRIDE;
  }
  if (r->data.shape[0] != N || r->data.shape[1] != H || r->data.shape[2] != S) return RK_ERR_SHAPE;
  return S < (INT64_C(1) << 30) ? RK_OK : RK_ERR_SHAPE;  // (rows that repeat by stride 0 can be any number)
}

int check_float(const rk_tensor* t, int ndim) {
  const int st = rk::check_desc(t, ndim);
  if (st) return st;
  return rk::is_float_param(t->dtype) ? RK_OK : RK_ERR_DTYPE;
}

int make_plan(const Call& c, int cus, Plan* out) {
  Plan p;
  memset(&p, 0, sizeof(p));
  int st = check_float(c.q, 3);
  if (st) return st;
  if (!c.k[kFull] || !c.v[kFull]) return RK_ERR_NULL;
  p.B = c.q->shape[0];
  p.Hq = c.q->shape[1];
  p.D = c.q->shape[2];
  if (p.D < 1 || p.D > 128) return RK_ERR_HEAD_DIM;
  if (c.groups <= 0) return RK_ERR_ARG;
  p.G = c.groups;
  p.H = c.k[kFull]->data.ndim == 4 ? c.k[kFull]->data.shape[1] : 0;
  if (p.H <= 0 || p.G > p.Hq || p.Hq % p.G != 0 || p.H != p.Hq / p.G) return RK_ERR_HEADS;
  p.format = c.k[kFull]->format;
  if (p.format != RK_ROWS_PLAIN && p.format != RK_ROWS_MX8 && p.format != RK_ROWS_MX4) return RK_ERR_ARG;
  const bool quantised = p.format != RK_ROWS_PLAIN;
  if (!quantised && (!c.shared || !rk::is_half(c.q->dtype))) return RK_ERR_DTYPE;
  const int64_t N = c.shared ? 1 : p.B;
  bool have[kSpans];
  for (int i = 0; i < kSpans; ++i) {
    have[i] = c.k[i] != nullptr;
    if (have[i] != (c.v[i] != nullptr)) return RK_ERR_NULL;
    if (have[i] && c.k[i]->data.ndim != 4) return RK_ERR_RANK;
    p.S[i] = have[i] ? c.k[i]->data.shape[2] : 0;
  }
  if (have[kRotated]) {
    if (!c.R) return RK_ERR_NULL;
    if ((st = check_float(c.R, 4))) return st;
    p.Dk = c.R->shape[3];
    if (p.Dk < 0 || p.Dk > p.D) return RK_ERR_KEEP_DIM;
    if (c.R->shape[0] != N || c.R->shape[1] != p.H || c.R->shape[2] != p.D) return RK_ERR_SHAPE;
    if (c.dm) {
      if ((st = check_float(c.dm, 3))) return st;
      if (c.dm->shape[0] != N || c.dm->shape[1] != p.H || c.dm->shape[2] != p.D) return RK_ERR_SHAPE;
    }
  }
  p.vec = true;
  for (int i = 0; i < kSpans; ++i) {
    if (!have[i]) continue;
    const int64_t n = i == kTail ? p.B : N;
    if ((st = check_rows(c.k[i], p.format, c.q->dtype, n, p.H, p.S[i], i == kRotated ? p.Dk : p.D))) return st;
    if ((st = check_rows(c.v[i], p.format, c.q->dtype, n, p.H, p.S[i], p.D))) return st;
    if (!quantised && p.S[i] > 0) {
      const bool keys = i != kRotated || p.Dk > 0;
      p.vec = p.vec && rk::vec_ok(&c.v[i]->data) && p.D % 8 == 0 &&
              (!keys || (rk::vec_ok(&c.k[i]->data) && c.k[i]->data.shape[3] % 8 == 0));
    }
  }
  if (c.mask) {
    if ((st = rk::check_desc(c.mask, 2))) return st;
    if (c.mask->dtype != RK_U8) return RK_ERR_DTYPE;
    if (c.mask->shape[0] != p.B || c.mask->shape[1] != p.S[kFull]) return RK_ERR_SHAPE;
  }
  if (c.out) {
    if ((st = rk::check_desc(c.out, 3))) return st;
    if (c.out->dtype != c.q->dtype) return RK_ERR_DTYPE;
    for (int i = 0; i < 3; ++i) {
      if (c.out->shape[i] != c.q->shape[i]) return RK_ERR_SHAPE;
      if (c.out->shape[i] > 1 && c.out->stride[i] == 0) return RK_ERR_STRIDE;  // two rows at one address
    }
  }

  p.kf = p.D <= 64 ? 2 : 4;
  p.kv = p.S[kRotated] == 0 ? 0 : p.Dk <= 32 ? 1 : p.Dk <= 64 ? 2 : 4;
  p.terms = quantised ? (c.q->dtype == RK_F32 ? 3 : 2) : 1;
  if (p.B >= kMaxGrid / p.Hq) return RK_ERR_SHAPE;
  p.rows = p.B * p.Hq;
  int64_t cost[kSpans], shared_bytes = 0, shared_tokens = 0;  // cost: bytes of a token
  for (int i = 0; i < kSpans; ++i) {
    const int64_t kd = i == kRotated ? p.Dk : p.D;
    cost[i] = quantised ? rk::mx_row_bytes(kd, p.format) + rk::mx_row_bytes(p.D, p.format) : 2 * (kd + p.D);
    if (i == kTail) continue;
    shared_bytes += p.S[i] * cost[i];
    shared_tokens += p.S[i];
  }
  p.tile = c.shared && p.vec && p.terms < 3 && shared_tokens > 0 &&
           cdiv(p.B * p.G, 16) * shared_bytes >= kTileBytes * shared_tokens;
  p.join = p.tile && p.S[kTail] > 0 && p.S[kTail] <= kJoinTokens;
  int64_t total = 0;
  for (int i = 0; i < kSpans; ++i) {
    const bool per_request = !c.shared || i == kTail;
    p.blocks[i] = cdiv(per_request ? p.G : p.B * p.G, p.tile && i != kTail ? 64 : 16);
    p.units[i] = p.H * p.blocks[i] * (per_request ? p.B : 1);
    if (p.units[i] * p.S[i] >= (INT64_C(1) << 50)) return RK_ERR_SHAPE;
    if (!(p.tile && i == kTail)) total += p.units[i] * p.S[i] * cost[i];
  }
  // Equal shares of the bytes for every workgroup, of whole rounds of the
  // workgroups that are resident at a time: the fewest rounds that keep a
  // share at kMaxShare, and within them the largest grid that fits.  Spans that
  // are not split fill slots by their bytes, short ones many to a slot (as many
  // slots as workgroups would leave the others too few: 16 requests of 8 heads
  // with 264 tokens behind 8192, 34.0 us and 30.6); tiles fill one each.
  auto split = [&](int64_t slots) {
    const int64_t rounds = std::max<int64_t>(cdiv(total, slots * kMaxShare), 1);
    const int64_t align = rk::kSpanWaves * rk::kSpanBlk;
    for (int64_t share = std::max<int64_t>(cdiv(total, slots * rounds), 1);; share += cdiv(share, 32)) {
      p.np = 0;
      int64_t used = 0;
      bool least = true;  // one workgroup per unit and span
      for (int i = 0; i < kSpans; ++i) {
        p.wgs[i] = p.chunk[i] = 0;
        if (p.S[i] == 0 || (p.join && i == kTail)) continue;
        p.chunk[i] = std::min(round_up(cdiv(share, cost[i]), align), round_up(p.S[i], align));
        p.wgs[i] = cdiv(p.S[i], p.chunk[i]);
        p.np += p.wgs[i];
        if (p.tile && i == kTail) continue;  // a launch of its own
        least = least && p.wgs[i] == 1;
        used += p.wgs[i] > 1 || p.tile ? p.wgs[i] * p.units[i] : cdiv(p.units[i] * p.S[i] * cost[i], share);
      }
      if (least || used <= slots * rounds) break;
    }
  };
  // Three workgroups a CU (16 requests of 7 heads on a KV head over 32768 4-bit
  // rows: 46.2 us, 48.3 with four, 49.9 with two; 32 requests of one head to 16000
  // 8-bit rows: 436, 431, 436).  Over 64 queries a workgroup's
  // records weigh as much as 64 tokens' rows and the join reads them again: two
  // there where three would leave it less than 768 tokens (32 requests of 4 heads
  // behind 16001: 35 us at two, chunks of 512 tokens, 38 at three, of 384; 64 of 7
  // heads behind 32768: 81 at two, 73 at three, of 1200; between them nothing was
  // measured).
  split((int64_t)cus * 3);
  if (p.tile && std::max(p.chunk[kRotated], p.chunk[kFull]) < 768) split((int64_t)cus * 2);
  if (p.join) {
    p.chunk[kTail] = round_up(p.S[kTail], rk::kSpanWaves * rk::kSpanBlk);
    p.wgs[kTail] = 1;
  }
  int64_t ids = 0;
  for (int i = 0; i < kSpans; ++i) ids += launched(p, i);
  if (ids >= kMaxGrid || p.rows * p.np >= (INT64_C(1) << 40)) return RK_ERR_SHAPE;
  const int64_t dv = p.kf == 2 ? 64 : 128;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return here;
  };
  // Queries as the split launch takes them: eight channels in one aligned
  // piece; their rotation there if everything has q's 16-bit type and lies in
  // pieces as well, else in a launch ahead.
  p.copy_q = !rk::vec_ok(c.q) || p.D % 8 != 0;
  p.ahead = p.kv && (p.copy_q || c.q->dtype == RK_F32 || p.Dk == 0 || p.Dk % 8 != 0 || c.R->dtype != c.q->dtype ||
                     !rk::vec_ok(c.R) || (c.dm && (c.dm->dtype != c.q->dtype || !rk::vec_ok(c.dm))));
  const size_t el = c.q->dtype == RK_F32 ? 4 : 2;
  p.q = take(p.copy_q ? (size_t)p.rows * round_up(p.D, 8) * el : 0);
  p.qr = take(p.ahead ? (size_t)p.rows * std::max(p.terms, 2) * 32 * p.kv * 2 : 0);
  p.bias = take(p.ahead ? (size_t)p.rows * 4 : 0);
  p.qtop = take(p.ahead && !quantised && c.q->dtype == RK_F16 ? (size_t)p.rows * 4 : 0);
  // rotated rows without channels: one zero row and its scales
  p.zero_bytes = p.kv && p.Dk == 0 ? 256 + (size_t)round_up(p.S[kRotated], 32) : 0;
  p.zero = take(p.zero_bytes);
  p.acc = take((size_t)(p.rows * p.np) * dv * 4);
  p.ml = take((size_t)(p.rows * p.np) * 8);
  p.total = at;
  *out = p;
  return RK_OK;
}

int null_data(const Call& c, const Plan& p) {
  if (!c.q->data || !c.out || !c.out->data) return RK_ERR_NULL;
  for (int i = 0; i < kSpans; ++i) {
    if (p.S[i] == 0) continue;
    if (!c.v[i]->data.data || (p.format != RK_ROWS_PLAIN && !c.v[i]->scales.data)) return RK_ERR_NULL;
    if (i == kRotated && p.Dk == 0) continue;
    if (!c.k[i]->data.data || (p.format != RK_ROWS_PLAIN && !c.k[i]->scales.data)) return RK_ERR_NULL;
  }
  if (p.kv && p.Dk > 0 && !c.R->data) return RK_ERR_NULL;
  if (p.kv && c.dm && !c.dm->data) return RK_ERR_NULL;
  if (c.mask && p.S[kFull] > 0 && !c.mask->data) return RK_ERR_NULL;
  return RK_OK;
}

Span make_span(const Call& c, const Plan& p, int i, char* ws) {
  const rk_rows *k = c.k[i], *v = c.v[i];
  Span s;
  memset(&s, 0, sizeof(s));
  const bool quantised = p.format != RK_ROWS_PLAIN;
  s.v = v->data.data;
  s.v_sb = v->data.stride[0]; s.v_sh = v->data.stride[1];
  s.v_ss = (uint32_t)v->data.stride[2]; s.v_sd = (uint32_t)v->data.stride[3];
  if (i == kRotated && p.Dk == 0) {
    s.k = ws + p.zero;
    s.ksc = (const uint8_t*)(ws + p.zero + 256);
    s.k_sd = 1;
  } else {
    s.k = k->data.data;
    s.k_sb = k->data.stride[0]; s.k_sh = k->data.stride[1];
    s.k_ss = (uint32_t)k->data.stride[2]; s.k_sd = (uint32_t)k->data.stride[3];
    s.width = (int32_t)(quantised ? rk::mx_width(k->head_dim) : k->head_dim);
    if (quantised) {
      s.ksc = (const uint8_t*)k->scales.data;
      s.ksc_sb = k->scales.stride[0]; s.ksc_sh = k->scales.stride[1]; s.ksc_sn = (uint32_t)k->scales.stride[2];
    }
  }
  if (quantised) {
    s.vsc = (const uint8_t*)v->scales.data;
    s.vsc_sb = v->scales.stride[0]; s.vsc_sh = v->scales.stride[1]; s.vsc_sn = (uint32_t)v->scales.stride[2];
  }
  s.len = c.len[i];
  if (i == kFull && c.mask) {
    s.mask = (const uint8_t*)c.mask->data;
    s.m_sb = c.mask->stride[0]; s.m_ss = c.mask->stride[1];
  }
  s.S = (int32_t)p.S[i];
  s.chunk = (int32_t)p.chunk[i];
  s.wgs = (int32_t)p.wgs[i];
  return s;
}

int resolve_cus(int num_cus, int* st) {
  *st = RK_OK;
  if (num_cus > 0) return num_cus;
  const int cus = num_cus < 0 ? 0 : rk::current_device_cus(nullptr);
  if (cus <= 0) *st = num_cus < 0 ? RK_ERR_ARG : RK_ERR_NO_DEVICE;
  return cus;
}

int run(const Call& c, void* workspace, size_t workspace_bytes, void* stream) {
  Plan p;
  // everything but the split is checked before a device is asked for
  int st = make_plan(c, 1, &p);
  if (st) return st;
  if (!c.out) return RK_ERR_NULL;
  if (p.B == 0) return RK_OK;
  if ((st = null_data(c, p))) return st;
  const int cus = resolve_cus(0, &st);
  if (st) return st;
  if ((st = make_plan(c, cus, &p))) return st;
  if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < p.total) return RK_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  SpanArgs a;
  memset(&a, 0, sizeof(a));
  int64_t first = 0, np0 = 0;
  for (int i = 0; i < kSpans; ++i) {
    a.first[i] = (int32_t)first;
    a.heads[i] = (int32_t)std::max<int64_t>(p.units[i] / std::max<int64_t>(p.blocks[i], 1), 1);
    a.blocks[i] = (int32_t)std::max<int64_t>(p.blocks[i], 1);
    if (p.S[i] == 0) continue;
    a.span[i] = make_span(c, p, i, ws);
    a.span[i].np0 = (int32_t)np0;
    if (p.join && i == kTail) continue;
    first += launched(p, i);
    np0 += p.wgs[i];
  }
  const hipStream_t s = (hipStream_t)stream;
  hipError_t e = hipSuccess;
  a.q = c.q->data;
  a.q_sb = c.q->stride[0]; a.q_sh = c.q->stride[1];
  a.q_dtype = c.q->dtype;
  if (p.copy_q || p.ahead) {
    rk::QueryArgs qa;
    memset(&qa, 0, sizeof(qa));
    qa.q = c.q->data;
    qa.q_sb = c.q->stride[0]; qa.q_sh = c.q->stride[1]; qa.q_sd = c.q->stride[2];
    qa.q_dtype = c.q->dtype;
    qa.Hq = (int32_t)p.Hq; qa.G = (int32_t)p.G; qa.D = (int32_t)p.D; qa.Dp = (int32_t)round_up(p.D, 8);
    qa.shared = c.shared;
    if (p.copy_q) {
      qa.q_out = ws + p.q;
      a.q = ws + p.q;
      a.q_sb = p.Hq * qa.Dp; a.q_sh = qa.Dp;
    }
    if (p.ahead) {
      qa.R = c.R->data;
      qa.R_sb = c.R->stride[0]; qa.R_sh = c.R->stride[1]; qa.R_sd = c.R->stride[2]; qa.R_sk = c.R->stride[3];
      qa.r_dtype = c.R->dtype;
      if (c.dm) {
        qa.dm = c.dm->data;
        qa.dm_sb = c.dm->stride[0]; qa.dm_sh = c.dm->stride[1]; qa.dm_sd = c.dm->stride[2];
        qa.dm_dtype = c.dm->dtype;
      }
      qa.Dk = (int32_t)p.Dk; qa.W = 32 * p.kv; qa.terms = std::max(p.terms, 2);
      qa.f16 = p.format == RK_ROWS_PLAIN && c.q->dtype == RK_F16;
      qa.qr = (uint16_t*)(ws + p.qr);
      qa.bias = (float*)(ws + p.bias);
      a.qr = qa.qr;
      a.bias = qa.bias;
      if (qa.f16) a.qtop = qa.qtop = (float*)(ws + p.qtop);
    }
    hipLaunchKernelGGL(span_queries_kernel, dim3((unsigned)p.rows), dim3(128), 0, s, qa);
    if (hipGetLastError() != hipSuccess) return RK_ERR_HIP;
  }
  a.out = c.out->data;
  a.o_sb = c.out->stride[0]; a.o_sh = c.out->stride[1]; a.o_sd = c.out->stride[2];
  a.o_dtype = c.out->dtype;
  a.acc = (float*)(ws + p.acc);
  a.ml = (float*)(ws + p.ml);
  a.B = (int32_t)p.B; a.Hq = (int32_t)p.Hq; a.H = (int32_t)p.H; a.G = (int32_t)p.G;
  a.D = (int32_t)p.D; a.Dk = (int32_t)p.Dk; a.np = (int32_t)p.np;
  a.shared = c.shared;
  a.scale_log2 = rk::kLog2e / sqrtf((float)p.D);
  if (p.zero_bytes) {
    hipLaunchKernelGGL(span_zero_kernel, dim3(64), dim3(256), 0, s, (uint32_t*)(ws + p.zero),
                       (int64_t)(p.zero_bytes / 4));
    if (hipGetLastError() != hipSuccess) return RK_ERR_HIP;
  }
  if (p.kv && !p.ahead) {
    a.R = c.R->data;
    a.R_sb = c.R->stride[0]; a.R_sh = c.R->stride[1]; a.R_sd = c.R->stride[2];
    if (c.dm) {
      a.dm = c.dm->data;
      a.dm_sb = c.dm->stride[0]; a.dm_sh = c.dm->stride[1];
    }
  }
  auto split = [&](const SpanArgs& b, int kv, int64_t grid) {
    if (p.format == RK_ROWS_MX8) return rk::span_launch_mx8(kv, p.kf, p.terms, b, (unsigned)grid, s);
    if (p.format == RK_ROWS_MX4) return rk::span_launch_mx4(kv, p.kf, p.terms, b, (unsigned)grid, s);
    if (c.q->dtype == RK_F16) return rk::span_launch_f16(kv, p.kf, p.vec, b, (unsigned)grid, s);
    return rk::span_launch_bf16(kv, p.kf, p.vec, b, (unsigned)grid, s);
  };
  if (!p.tile) {
    if (first > 0 && split(a, p.kv, first) != hipSuccess) return RK_ERR_HIP;
  } else {
    const int64_t shared = a.first[kTail];
    if (first > shared) {  // a suffix that is split: a launch of its own
      SpanArgs tail = a;
      tail.first[kRotated] = tail.first[kFull] = tail.first[kTail] = 0;
      if (split(tail, 0, first - shared) != hipSuccess) return RK_ERR_HIP;
    }
    const unsigned grid = (unsigned)shared;
    if (p.format == RK_ROWS_MX8)
      e = rk::tile_launch_mx8(p.kv, p.kf, a, grid, s);
    else if (p.format == RK_ROWS_MX4)
      e = rk::tile_launch_mx4(p.kv, p.kf, a, grid, s);
    else if (c.q->dtype == RK_F16)
      e = rk::tile_launch_f16(p.kv, p.kf, a, grid, s);
    else
      e = rk::tile_launch_bf16(p.kv, p.kf, a, grid, s);
    if (e != hipSuccess) return RK_ERR_HIP;
  }
  if (p.join) {
    const unsigned grid = (unsigned)launched(p, kTail);
    if (p.format == RK_ROWS_MX8)
      e = rk::span_join_mx8(p.kf, a, grid, s);
    else if (p.format == RK_ROWS_MX4)
      e = rk::span_join_mx4(p.kf, a, grid, s);
    else if (c.q->dtype == RK_F16)
      e = rk::span_join_f16(p.kf, a, grid, s);
    else
      e = rk::span_join_bf16(p.kf, a, grid, s);
    return e == hipSuccess ? RK_OK : RK_ERR_HIP;
  }
  const int w = p.np > kMergeWave ? 4 : 1;
  const dim3 mg((unsigned)cdiv(p.rows, 4 / w));
  if (p.kf == 2 && w == 1)
    hipLaunchKernelGGL((span_merge_kernel<64, 1>), mg, dim3(256), 0, s, a);
  else if (p.kf == 2)
    hipLaunchKernelGGL((span_merge_kernel<64, 4>), mg, dim3(256), 0, s, a);
  else if (w == 1)
    hipLaunchKernelGGL((span_merge_kernel<128, 1>), mg, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((span_merge_kernel<128, 4>), mg, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_HIP;
}

int check_call(const Call& c, int32_t num_cus, size_t* bytes) {
  Plan p;
  int st = make_plan(c, 1, &p);
  if (st) return st;
  const int cus = resolve_cus(num_cus, &st);
  if (st) return st;
  if ((st = make_plan(c, cus, &p))) return st;
  if (bytes) *bytes = p.total;
  return RK_OK;
}

Call quantized_call(const rk_tensor* q, const rk_tensor* R, const rk_tensor* dm, const rk_rows* k_full,
                    const rk_rows* v_full, const rk_tensor* mask, const int32_t* len, const rk_rows* k_sparse,
                    const rk_rows* v_sparse, int64_t groups, const rk_tensor* out) {
  Call c;
  memset(&c, 0, sizeof(c));
  c.q = q; c.R = R; c.dm = dm; c.mask = mask; c.out = out;
  c.k[kFull] = k_full; c.v[kFull] = v_full; c.len[kFull] = len;
  c.k[kRotated] = k_sparse; c.v[kRotated] = v_sparse;
  c.groups = groups;
  return c;
}

Call shared_call(const rk_tensor* q, const rk_tensor* R, const rk_tensor* dm, const rk_rows* k_prefix,
                 const rk_rows* v_prefix, const rk_rows* k_sparse, const rk_rows* v_sparse, const rk_rows* k_suffix,
                 const rk_rows* v_suffix, const int32_t* len, int64_t groups, const rk_tensor* out) {
  Call c = quantized_call(q, R, dm, k_prefix, v_prefix, nullptr, nullptr, k_sparse, v_sparse, groups, out);
  c.k[kTail] = k_suffix; c.v[kTail] = v_suffix; c.len[kTail] = len;
  c.shared = true;
  return c;
}

}  // namespace

extern "C" int rk_quantized_decode_check(const rk_tensor* q, const rk_tensor* R_partial, const rk_tensor* delta_mu,
                                         const rk_rows* k_full, const rk_rows* v_full, const rk_tensor* mask_full,
                                         const rk_rows* k_sparse, const rk_rows* v_sparse, int64_t num_kv_groups,
                                         const rk_tensor* out, int32_t num_cus, size_t* workspace_bytes) {
  return check_call(quantized_call(q, R_partial, delta_mu, k_full, v_full, mask_full, nullptr, k_sparse, v_sparse,
                                   num_kv_groups, out),
                    num_cus, workspace_bytes);
}

extern "C" int rk_quantized_decode(const rk_tensor* q, const rk_tensor* R_partial, const rk_tensor* delta_mu,
                                   const rk_rows* k_full, const rk_rows* v_full, const rk_tensor* mask_full,
                                   const int32_t* len_full, const rk_rows* k_sparse, const rk_rows* v_sparse,
                                   int64_t num_kv_groups, const rk_tensor* out, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  return run(quantized_call(q, R_partial, delta_mu, k_full, v_full, mask_full, len_full, k_sparse, v_sparse,
                            num_kv_groups, out),
             workspace, workspace_bytes, stream);
}

extern "C" int rk_shared_prefix_decode_check(const rk_tensor* q, const rk_tensor* R_partial, const rk_tensor* delta_mu,
                                             const rk_rows* k_prefix, const rk_rows* v_prefix, const rk_rows* k_sparse,
                                             const rk_rows* v_sparse, const rk_rows* k_suffix, const rk_rows* v_suffix,
                                             int64_t num_kv_groups, const rk_tensor* out, int32_t num_cus,
                                             size_t* workspace_bytes) {
  return check_call(shared_call(q, R_partial, delta_mu, k_prefix, v_prefix, k_sparse, v_sparse, k_suffix, v_suffix,
                                nullptr, num_kv_groups, out),
                    num_cus, workspace_bytes);
}

extern "C" int rk_shared_prefix_decode(const rk_tensor* q, const rk_tensor* R_partial, const rk_tensor* delta_mu,
                                       const rk_rows* k_prefix, const rk_rows* v_prefix, const rk_rows* k_sparse,
                                       const rk_rows* v_sparse, const rk_rows* k_suffix, const rk_rows* v_suffix,
                                       const int32_t* len_suffix, int64_t num_kv_groups, const rk_tensor* out,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  return run(shared_call(q, R_partial, delta_mu, k_prefix, v_prefix, k_sparse, v_sparse, k_suffix, v_suffix,
                         len_suffix, num_kv_groups, out),
             workspace, workspace_bytes, stream);
}
