// rk_span.h -- one token's attention over spans of plain or quantised rows:
// the argument block and launch geometry that the host code (rk_span.hip) and
// the per-format kernel units (rk_span_{f16,bf16,mx8,mx4}.hip) share.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace rk {

// One span of rows: K scores, V values, [B?, H_kv, S, *].  Strides in bytes
// for quantised rows, in elements for plain ones.
struct Span {
  const void* k;
  const void* v;
  const uint8_t* ksc;  // scales [B?, H_kv, blocks, S'] of quantised rows
  const uint8_t* vsc;
  const int32_t* len;   // rows t < len[b] count (optional)
  const uint8_t* mask;  // rows with mask[b, t] != 0 count (optional)
  int64_t k_sb, k_sh, v_sb, v_sh;
  int64_t ksc_sb, ksc_sh, vsc_sb, vsc_sh;
  int64_t m_sb, m_ss;
  uint32_t k_ss, k_sd, v_ss, v_sd;  // within a head: < 2^31 in all
  uint32_t ksc_sn, vsc_sn;
  int32_t S, chunk;  // tokens; tokens per workgroup
  int32_t wgs;       // workgroups of a unit
  int32_t np0;       // record number of the unit's first workgroup
  int32_t width;     // stored channels of a score row (a multiple of 32, or D)
};

// Spans by what their rows score with.
enum { kRotated = 0, kFull = 1, kTail = 2, kSpans = 3 };

struct SpanArgs {
  Span span[kSpans];
  // units: (b, kv, row block) or, where the batch shares the span's rows,
  // (kv, row block over the batch's queries)
  int32_t heads[kSpans], blocks[kSpans];  // heads: (b, kv) or kv; blocks: row blocks of each
  int32_t first[kSpans];  // first workgroup of each span
  const void* q;       // [B, H_q, *] in whole, 16-byte aligned pieces of eight channels
  void* out;
  const uint16_t* qr;  // rotated queries formed ahead, [row][terms][32 KV] 16 bits, or null
  const float* bias;   // ... and q . delta_mu
  float* acc;  // [row][np][DV] partial sums
  float* ml;   // [row][np][2] running maximum and sum
  int64_t q_sb, q_sh, o_sb, o_sh, o_sd;
  int32_t B, Hq, H, G, D, Dk, np, shared;
  int32_t q_dtype, o_dtype;
  float scale_log2;  // log2(e) / sqrt(D)
  // the rotation of the rotated span's queries (qr null): in q's 16-bit type,
  // unit column stride, aligned pieces of eight channels
  const void* R;
  const void* dm;
  int64_t R_sb, R_sh, R_sd, dm_sb, dm_sh;
  const float* qtop;  // with qr of fp16 terms: a row's largest |q R|
};

// Queries that the split launch does not take as they are: a copy of q in
// whole pieces, and q R in `terms` terms with q . delta_mu.
struct QueryArgs {
  const void* q;
  const void* R;
  const void* dm;
  void* q_out;      // [row][Dp], or null
  uint16_t* qr;     // [row][terms][W], or null
  float* bias;
  float* qtop;      // [row], fp16 terms' alone
  int64_t q_sb, q_sh, q_sd, R_sb, R_sh, R_sd, R_sk, dm_sb, dm_sh, dm_sd;
  int32_t Hq, G, D, Dp, Dk, W, terms, shared, q_dtype, r_dtype, dm_dtype, f16;
};

constexpr int kSpanThreads = 256;
constexpr int kSpanWaves = 4;
constexpr int kSpanBlk = 32;  // tokens of a wave's step

// fp16 terms of q R.  fp16 ends at 65504, and queries of order 10^4 take q R past
// it: a row whose largest entry `top` is 2^15 or more is split as q R 2^-shift,
// below 2^15, and its scores take 2^shift back in their factor.  Both are exact.
// (Each row by itself: a large query leaves its neighbours' terms alone.)
constexpr float kSplitTop = 32768.f;
__device__ __forceinline__ int split_shift(float top) {
  return top >= kSplitTop && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
}

// The split launch: kv = score blocks of 32 channels of the rotated span (0:
// none, 1, 2 or 4), kf the full-width spans' (2: D <= 64, or 4), terms = 16-bit
// terms that a query is exact in.
hipError_t span_launch_f16(int kv, int kf, bool vec, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t span_launch_bf16(int kv, int kf, bool vec, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t span_launch_mx8(int kv, int kf, int terms, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t span_launch_mx4(int kv, int kf, int terms, const SpanArgs& a, unsigned grid, hipStream_t s);

// The split launch over rows that many queries share, 64 of them a workgroup
// (rk_tile_dev.h; 16-bit queries, whole pieces).
hipError_t tile_launch_f16(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t tile_launch_bf16(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t tile_launch_mx8(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t tile_launch_mx4(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s);

// The launch behind that one: the suffix rows and the join of all records.
hipError_t span_join_f16(int kf, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t span_join_bf16(int kf, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t span_join_mx8(int kf, const SpanArgs& a, unsigned grid, hipStream_t s);
hipError_t span_join_mx4(int kf, const SpanArgs& a, unsigned grid, hipStream_t s);

}  // namespace rk
