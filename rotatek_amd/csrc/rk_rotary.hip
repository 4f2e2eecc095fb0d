// rk_rotary.hip -- rotation by position and the append to a paged cache on
// MI355X (gfx950): rk_rotary, rk_paged_append of rotatek_hip.h.
//
// Mathematics.  Pair i of a head (channels i and i + P) turns by
// a = pos[axis(i)] f[i].  pos f is formed in 64 bits, where it is exact to
// 2^-53, and so are its turns a / 2 pi, of which only the fraction is kept: at
// position 10^5 an angle in 32 bits is off by 2^-8.  Its sine and cosine are formed
// in 64 bits too and rounded once, to 32: they are few, one a token and pair for all
// heads (3 x 32 heads x 2304 tokens of 80 channels in fp32: 26.4 us, 26.1 with 32-bit
// ones, which leave twice the error; all others as long).  A pair is rounded as it
// is stored.
//
// A workgroup takes a few tokens.  Each pair's sine and cosine are formed once
// for all heads of the token and go through LDS; then every lane turns a
// vector of pairs (16 bytes from either half of the head) of one head.  In an
// append the same pass writes Keys and Values to their pages.
//
// The bytes bound it: 1.6 GB of video heads in 300 us, 5.3 TB/s; a plain copy reaches
// 6.3 at best (a piece of 16 bytes a thread), 5.8 with four pieces.
#include <hip/hip_runtime.h>
#include <string.h>

#include <algorithm>

#include "rk_common.h"
#include "rk_host.h"
#include "rk_paged.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 2;  // tokens of a workgroup, a wave each where their places are found
constexpr int kMaxPairs = 64;
constexpr int kMaxAxes = 4;

enum { kQ = 0, kK = 1, kV = 2, kParts = 3 };

struct Part {
  const void* x;
  void* y;
  int64_t x_sb, x_sh, x_ss, x_sd;  // elements; token (b, t)
  int64_t y_sb, y_sh, y_ss, y_sd;  // ... of a page, a head, a row where the token goes to its page
  int32_t heads;
};

// i / d for the i that occur: by a product where that is exact.
struct Divisor {
  uint32_t d, magic;
  __device__ __forceinline__ int quotient(int i) const {
    return magic ? (int)__umulhi((uint32_t)i, magic) : (int)((uint32_t)i / d);
  }
};
Divisor divisor_of(int64_t d, int64_t below) {
  // 2^32 / d rounded up, by m: i m / 2^32 is off by less than i d / 2^32 of 1 / d
  return {(uint32_t)d, d > 1 && below * d < (INT64_C(1) << 32) ? (uint32_t)((INT64_C(1) << 32) / d + 1) : 0u};
}

struct RotaryArgs {
  Part part[kParts];
  // Work of a token: for each head items of two vectors, `turned` that turn (from
  // either half of the pairs) and the others that are copied.
  int32_t turned, copied, all, nq, nk;
  Divisor token, head[kParts];
  const void* pos;  // null: nothing turns
  const float* freq;
  int64_t p_sa, p_sb, p_st, f_s;
  uint32_t axis[4];  // two bits a pair
  int32_t pos64;
  float sign;
  int32_t P, D;
  int32_t T;  // tokens of a batch row
  int64_t N;  // tokens
  int32_t tokens;  // of a workgroup
  // the pages (paged)
  rk::PageMap map;
};

// cos and sin of so many turns, rounded once to 32 bits.
__device__ __forceinline__ float2 turn_of(double turns) {
  double s, c;
  sincospi(2.0 * (turns - __builtin_rint(turns)), &s, &c);
  return make_float2((float)c, (float)s);
}

// A pair turned.  The products are told apart (one rounded, one fused), so that
// every path gives the same bits.
__device__ __forceinline__ float2 turn(float lo, float hi, float2 cs) {
  return make_float2(__builtin_fmaf(lo, cs.x, -(hi * cs.y)), __builtin_fmaf(hi, cs.x, lo * cs.y));
}

// rk::request_of by a wave.
__device__ __forceinline__ int request_of_wave(const rk::PageMap& m, int64_t n) {
  const int lane = threadIdx.x & 63;
  int low = 0, left = m.B;
  while (left > 1) {
    const int step = (left + 63) / 64, at = lane * step;
    const uint64_t before = __ballot(at < left && m.starts[low + min(at, left - 1)] <= n);
    const int up = before ? 63 - __builtin_clzll(before) : 0;
    low += up * step;
    left = min(step, left - up * step);
  }
  return low;
}

// rk::place_of by a wave: what up to 64 requests say in one read instead of three
// that wait for each other (32 requests of one token each: 5.2 us, 5.0 so).
__device__ __forceinline__ int64_t place_of_wave(const rk::PageMap& m, int64_t n, int* row) {
  if (!m.starts || m.B < 1 || m.B > 64) return rk::place_of(m, n, m.starts ? request_of_wave(m, n) : 0, row);
  const int lane = threadIdx.x & 63, i = min(lane, m.B - 1);
  const int s = m.starts[i], e = m.starts[i + 1], len = m.lens[i];
  const uint64_t before = __ballot(lane < m.B && s <= n);
  const int b = before ? 63 - __builtin_clzll(before) : 0;
  return rk::place_in(m, n, b, __builtin_amdgcn_readlane(s, b), __builtin_amdgcn_readlane(e, b),
                      __builtin_amdgcn_readlane(len, b), row);
}

// Token n is t of batch row b.
__device__ __forceinline__ void batch_row(const RotaryArgs& a, int64_t n, int64_t* b, int64_t* t) {
  *b = a.N >> 31 ? n / a.T : (uint32_t)n / (uint32_t)a.T;
  *t = n - *b * a.T;
}

// The part's of three (by selects: an indexed argument is a load of its own).
template <class V>
__device__ __forceinline__ V of(int which, V q, V k, V v) {
  return which == kQ ? q : which == kK ? k : v;
}

// E: elements at a time, up to 16 bytes.  PAGED: K and V go to their pages.
// ONCE: past the caches.
template <class DT, int E, bool PAGED, bool ONCE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const RotaryArgs a) {
  constexpr bool VEC = E > 1;
  constexpr int W = VEC ? E * DT::kBytes / 4 : 1;  // words of a vector
  typedef uint32_t vec __attribute__((ext_vector_type(W)));
  using word = typename std::conditional<DT::kBytes == 4, uint32_t, uint16_t>::type;
  __shared__ float2 s_turn[kMaxTokens * kMaxPairs];
  __shared__ const word* s_x[kMaxTokens][kParts];  // a token's first element
  __shared__ word* s_y[kMaxTokens][kParts];        // null: nowhere
  const int tid = threadIdx.x;
  const int64_t n0 = (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)min((int64_t)a.tokens, a.N - n0);
  if (a.pos) {
    for (int i = tid; i < tokens * a.P; i += kThreads) {
      const int tok = i / a.P, p = i - tok * a.P;
      int64_t b, t;
      batch_row(a, n0 + tok, &b, &t);
      const int axis = (a.axis[p >> 4] >> (2 * (p & 15))) & 3;
      const int64_t at = axis * a.p_sa + b * a.p_sb + t * a.p_st;
      const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
      float2 cs = turn_of(pos * (double)a.freq[p * a.f_s] * 0.15915494309189533577);
      cs.y *= a.sign;
      s_turn[tok * kMaxPairs + p] = cs;
    }
  }
  if constexpr (PAGED) {
    // a wave finds a token's place, the last ones as the first have the angles (32
    // requests of one token each: 5.0 us by the first, 4.2 so; prompts 171 and 165)
    const int tok = kThreads / 64 - 1 - __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tok < tokens) {
      int row = 0;
      const int64_t page = place_of_wave(a.map, n0 + tok, &row);
      if ((tid & 63) == 0) {
        for (int which : {kK, kV})
          s_y[tok][which] = page < 0 ? nullptr : (word*)a.part[which].y + page * a.part[which].y_sb + row * a.part[which].y_ss;
      }
    }
  }
  if (tid < tokens * kParts) {
    const int tok = tid / kParts, which = tid - tok * kParts;
    const Part& p = a.part[which];
    int64_t b, t;
    batch_row(a, n0 + tok, &b, &t);
    s_x[tok][which] = (const word*)p.x + b * p.x_sb + t * p.x_ss;
    if (!PAGED || which == kQ) s_y[tok][which] = (word*)p.y + b * p.y_sb + t * p.y_ss;
  }
  __syncthreads();
  // (addresses that come from LDS: which memory they are in has to be said)
  typedef __attribute__((address_space(1))) word global_word;
  typedef __attribute__((address_space(1))) vec global_vec;
  const int per_token = a.token.d;
  for (int i = tid; i < tokens * per_token; i += kThreads) {
    const int tok = a.token.quotient(i);
    int u = i - tok * per_token;
    const int which = u < a.nq ? kQ : u < a.nq + a.nk ? kK : kV;
    u -= which == kQ ? 0 : which == kK ? a.nq : a.nq + a.nk;
    const Part &pq = a.part[kQ], &pk = a.part[kK], &pv = a.part[kV];
    const Divisor d = which == kV ? a.head[kV] : a.head[kQ];
    const int h = d.quotient(u), item = u - h * (int)d.d;
    if (PAGED && !s_y[tok][which]) continue;
    global_word* y = (global_word*)s_y[tok][which] + h * of(which, pq.y_sh, pk.y_sh, pv.y_sh);
    const global_word* x = (const global_word*)s_x[tok][which] + h * of(which, pq.x_sh, pk.x_sh, pv.x_sh);
    const bool turns = which != kV && item < a.turned;
    // the item's vectors: channels c and c2 (copied: if that is below D)
    const int first = which == kV ? 0 : a.turned, n = which == kV ? a.all : a.copied, half = (n + 1) / 2;
    const int base = which == kV || !a.pos ? 0 : 2 * a.P;
    const int c = turns ? item * E : base + (item - first) * E;
    const int c2 = turns ? c + a.P : c + half * E;
    const bool two = turns || item - first + half < n;
    if constexpr (VEC) {
      vec lo = *(const global_vec*)(x + c), hi = lo;
      if (two) hi = *(const global_vec*)(x + c2);
      if (turns) {
        const float2* cs = s_turn + tok * kMaxPairs + c;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const uint32_t wl = lo[e], wh = hi[e];
          if constexpr (DT::kBytes == 4) {
            const float2 y2 = turn(DT::to_f32(wl), DT::to_f32(wh), cs[e]);
            lo[e] = DT::from_f32(y2.x);
            hi[e] = DT::from_f32(y2.y);
          } else {
            const float2 y0 = turn(DT::to_f32((uint16_t)wl), DT::to_f32((uint16_t)wh), cs[2 * e]);
            const float2 y1 = turn(DT::to_f32((uint16_t)(wl >> 16)), DT::to_f32((uint16_t)(wh >> 16)), cs[2 * e + 1]);
            lo[e] = DT::pack2(y0.x, y1.x);
            hi[e] = DT::pack2(y0.y, y1.y);
          }
        }
      }
      if constexpr (ONCE) {
        __builtin_nontemporal_store(lo, (global_vec*)(y + c));
        if (two) __builtin_nontemporal_store(hi, (global_vec*)(y + c2));
      } else {
        *(global_vec*)(y + c) = lo;
        if (two) *(global_vec*)(y + c2) = hi;
      }
    } else {
      const int64_t x_sd = of(which, pq.x_sd, pk.x_sd, pv.x_sd), y_sd = of(which, pq.y_sd, pk.y_sd, pv.y_sd);
      word lo = x[c * x_sd], hi = lo;
      if (two) hi = x[c2 * x_sd];
      if (turns) {
        const float2 y2 = turn(DT::to_f32(lo), DT::to_f32(hi), s_turn[tok * kMaxPairs + c]);
        lo = DT::from_f32(y2.x);
        hi = DT::from_f32(y2.y);
      }
      y[c * y_sd] = lo;
      if (two) y[c2 * y_sd] = hi;
    }
  }
}

// The rotation's arguments: positions [A,B,T] or [A,N], frequencies [P], pairs
// of each axis.
int set_rotation(RotaryArgs* a, const rk_tensor* pos, const rk_tensor* freq, const int32_t* sections, int32_t axes,
                 int32_t interleaved, int32_t inverse, int64_t B, int64_t T, bool flat) {
  if (!pos || !freq || !sections) return RK_ERR_NULL;
  int st;
  if ((st = rk::check_desc(pos, flat ? 2 : 3)) || (st = rk::check_desc(freq, 1))) return st;
  if (pos->dtype != RK_I32 && pos->dtype != RK_I64) return RK_ERR_DTYPE;
  if (freq->dtype != RK_F32) return RK_ERR_DTYPE;
  if (axes < 1 || axes > kMaxAxes) return RK_ERR_ARG;
  if (interleaved < 0 || interleaved > 1 || inverse < 0 || inverse > 1) return RK_ERR_ARG;
  if (pos->shape[0] != axes) return RK_ERR_SHAPE;
  if (flat ? pos->shape[1] != T : pos->shape[1] != B || pos->shape[2] != T) return RK_ERR_SHAPE;
  const int64_t P = freq->shape[0];
  if (P < 1 || P > kMaxPairs || 2 * P > a->D) return RK_ERR_SHAPE;
  int64_t sum = 0;
  int32_t left[kMaxAxes];
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > P) return RK_ERR_ARG;
    left[i] = sections[i];
    sum += sections[i];
  }
  if (sum != P) return RK_ERR_ARG;
  int axis = 0;
  for (int i = 0; i < P; ++i) {
    while (!left[axis]) axis = (axis + 1) % axes;  // ends: P pairs are left in all
    a->axis[i >> 4] |= (uint32_t)axis << (2 * (i & 15));
    --left[axis];
    if (interleaved) axis = (axis + 1) % axes;
  }
  a->pos = pos->data;
  a->pos64 = pos->dtype == RK_I64;
  a->p_sa = pos->stride[0];
  a->p_sb = flat ? 0 : pos->stride[1];
  a->p_st = pos->stride[flat ? 1 : 2];
  a->freq = (const float*)freq->data;
  a->f_s = freq->stride[0];
  a->P = (int32_t)P;
  a->sign = inverse ? -1.f : 1.f;
  return RK_OK;
}

// Strides of [B,H,T,D], or of [N,H,D] as one batch row.
struct Strides {
  int64_t sb, sh, ss, sd;
};
Strides strides_of(const rk_tensor* t) {
  if (t->ndim == 4) return {t->stride[0], t->stride[1], t->stride[2], t->stride[3]};
  return {0, t->stride[1], t->stride[0], t->stride[2]};
}

void set_in(Part* p, const rk_tensor* x) {
  const Strides s = strides_of(x);
  p->x = x->data;
  p->x_sb = s.sb; p->x_sh = s.sh; p->x_ss = s.ss; p->x_sd = s.sd;
  p->heads = (int32_t)x->shape[1];
}
void set_out(Part* p, void* y, const Strides& s) {
  p->y = y;
  p->y_sb = s.sb; p->y_sh = s.sh; p->y_ss = s.ss; p->y_sd = s.sd;
}

// Elements that lie together and aligned in every row, up to 16 bytes of them.
int vector_of(const rk_tensor* t) {
  const int size = rk::dtype_size(t->dtype);
  int64_t n = 16 / size;
  if (t->stride[t->ndim - 1] != 1 && t->shape[t->ndim - 1] > 1) return 1;
  auto cut = [&](int64_t x) {
    while (n > 1 && x % n) n /= 2;
  };
  cut(t->shape[t->ndim - 1]);
  for (int i = 0; i < t->ndim - 1; ++i)
    if (t->shape[i] > 1) cut(t->stride[i]);
  while (n > 1 && (uintptr_t)t->data % (n * size)) n /= 2;
  return n * size < 4 ? 1 : (int)n;
}

// What a call writes must not repeat by a stride of 0.
bool distinct(const rk_tensor* t) {
  for (int i = 0; i < t->ndim; ++i)
    if (t->shape[i] > 1 && t->stride[i] == 0) return false;
  return true;
}

int check_x(const rk_tensor* x, int rank) {
  if (int st = rk::check_desc(x, rank)) return st;
  if (!rk::is_float_param(x->dtype)) return RK_ERR_DTYPE;
  const int64_t D = x->shape[rank - 1];
  if (D < 1 || D > 128) return RK_ERR_HEAD_DIM;
  return x->shape[1] >= (1 << 20) ? RK_ERR_HEADS : RK_OK;
}

bool same_shape(const rk_tensor* a, const rk_tensor* b) {
  if (a->ndim != b->ndim) return false;
  for (int i = 0; i < a->ndim; ++i)
    if (a->shape[i] != b->shape[i]) return false;
  return true;
}

// The same tokens and channels (heads may differ).
bool same_tokens(const rk_tensor* a, const rk_tensor* b) {
  if (a->ndim != b->ndim) return false;
  for (int i = 0; i < a->ndim; ++i)
    if (i != 1 && a->shape[i] != b->shape[i]) return false;
  return true;
}

template <class F>
int by_type(int dtype, int e, F&& f) {
  auto on = [&](auto dt) {
    constexpr int most = 16 / decltype(dt)::kBytes;
    if (e == most) return f(dt, std::integral_constant<int, most>{});
    if (e == most / 2) return f(dt, std::integral_constant<int, most / 2>{});
    if (e == most / 4 && most / 4 > 1) return f(dt, std::integral_constant<int, most / 4>{});
    f(dt, std::integral_constant<int, 1>{});
  };
  if (dtype == RK_F16)
    on(rk::F16{});
  else if (dtype == RK_BF16)
    on(rk::BF16{});
  else
    on(rk::F32{});
  return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_HIP;
}

// e: what all tensors allow.
template <bool PAGED>
int launch(RotaryArgs& a, int dtype, int e, void* stream) {
  while (a.pos && a.P % e) e /= 2;
  if (e * rk::dtype_size(dtype) < 4) e = 1;
  a.tokens = a.N >= 2048 ? kMaxTokens : 1;
  a.turned = a.pos ? a.P / e : 0;
  a.copied = (a.D - (a.pos ? 2 * a.P : 0)) / e;
  a.all = a.D / e;
  const int64_t per = a.turned + (a.copied + 1) / 2, half = (a.all + 1) / 2;
  const int64_t heads[kParts] = {a.part[kQ].heads, a.part[kK].heads, a.part[kV].heads};
  a.nq = (int32_t)(heads[kQ] * per);
  a.nk = (int32_t)(heads[kK] * per);
  const int64_t items = a.nq + a.nk + heads[kV] * half;
  a.token = divisor_of(items, kMaxTokens * items);
  a.head[kQ] = a.head[kK] = divisor_of(per, std::max(heads[kQ], heads[kK]) * per);
  a.head[kV] = divisor_of(half, heads[kV] * half);
  // Stores of whole lines leave the caches to others: 3 x 32 heads x 2304 tokens of
  // 80 channels in fp32 (142 MB in all) take 26 us (a copy of as much 23 at best), 39 with
  // ordinary stores; 17 prompts of up to 4097 tokens into pages 177 and
  // 183 (with places found behind the angles).  Lines
  // that two stores share have to meet in a cache: 23205 tokens of 96 heads of 96
  // channels in fp16 take 227 us with 48 pairs, 253 past the caches.
  const int size = rk::dtype_size(dtype), run = (a.pos ? a.P : a.D) * size;
  const bool once = e * size == 16 && run >= 128 && run % 32 == 0 && a.D * size % 32 == 0;
  const int64_t grid = (a.N + a.tokens - 1) / a.tokens;
  if (grid >= rk::kMostGroups) return RK_ERR_SHAPE;
  return by_type(dtype, e, [&](auto dt, auto n) {
    constexpr int E = decltype(n)::value;
    if constexpr (E * decltype(dt)::kBytes == 16)
      if (once) {
        hipLaunchKernelGGL((rotary_kernel<decltype(dt), E, PAGED, true>), dim3((unsigned)grid), dim3(kThreads), 0,
                           (hipStream_t)stream, a);
        return;
      }
    hipLaunchKernelGGL((rotary_kernel<decltype(dt), E, PAGED, false>), dim3((unsigned)grid), dim3(kThreads), 0,
                       (hipStream_t)stream, a);
  });
}

}  // namespace

extern "C" int rk_rotary(const rk_tensor* q, const rk_tensor* k, const rk_tensor* positions,
                         const rk_tensor* inv_freq, const int32_t* sections, int32_t axes, int32_t interleaved,
                         int32_t inverse, const rk_tensor* q_out, const rk_tensor* k_out, void* stream) {
  if (!q || !q_out || (k == nullptr) != (k_out == nullptr)) return RK_ERR_NULL;
  const int rank = q->ndim;
  if (rank != 3 && rank != 4) return RK_ERR_RANK;
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  int vec = 8;
  for (const rk_tensor* t : {q, q_out, k, k_out}) {
    if (!t) continue;
    if (int st = check_x(t, rank)) return st;
    if (t->dtype != q->dtype) return RK_ERR_DTYPE;
    if (!same_tokens(t, q)) return RK_ERR_SHAPE;
    vec = std::min(vec, vector_of(t));
  }
  if (!same_shape(q, q_out) || (k && !same_shape(k, k_out))) return RK_ERR_SHAPE;
  for (const rk_tensor* t : {q_out, k_out})
    if (t && !distinct(t)) return RK_ERR_STRIDE;
  a.D = (int32_t)q->shape[rank - 1];
  const int64_t B = rank == 4 ? q->shape[0] : 1, T = rank == 4 ? q->shape[2] : q->shape[0];
  if (T >= (INT64_C(1) << 31) || (T > 0 && B >= (INT64_C(1) << 40) / T)) return RK_ERR_SHAPE;
  if (int st = set_rotation(&a, positions, inv_freq, sections, axes, interleaved, inverse, B, T, rank == 3)) return st;
  a.T = (int32_t)T;
  a.N = B * T;
  set_in(&a.part[kQ], q);
  set_out(&a.part[kQ], q_out->data, strides_of(q_out));
  if (k) {
    set_in(&a.part[kK], k);
    set_out(&a.part[kK], k_out->data, strides_of(k_out));
  }
  if (a.N == 0 || a.part[kQ].heads + a.part[kK].heads == 0) return RK_OK;
  for (const Part& p : a.part)
    if (p.heads && (!p.x || !p.y)) return RK_ERR_NULL;
  if (!a.pos || !a.freq) return RK_ERR_NULL;
  return launch<false>(a, q->dtype, vec, stream);
}

extern "C" int rk_paged_append(const rk_tensor* k_new, const rk_tensor* v_new, const rk_pages* pages,
                               const int32_t* starts, const rk_tensor* q, const rk_tensor* q_out,
                               const rk_tensor* positions, const rk_tensor* inv_freq, const int32_t* sections,
                               int32_t axes, int32_t interleaved, void* stream) {
  if (!k_new || !v_new || !pages || (q == nullptr) != (q_out == nullptr)) return RK_ERR_NULL;
  if (q && !positions) return RK_ERR_NULL;
  const int rank = k_new->ndim;
  if (rank != 3 && rank != 4) return RK_ERR_RANK;
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  int64_t B = 0, cap = 0;
  int st = rk::set_pages(pages, &a.map, &B, &cap);
  if (st) return st;
  int vec = std::min(vector_of(&pages->k), vector_of(&pages->v));
  for (const rk_tensor* t : {k_new, v_new, q, q_out}) {
    if (!t) continue;
    if ((st = check_x(t, rank))) return st;
    if (t->dtype != k_new->dtype) return RK_ERR_DTYPE;
    if (!same_tokens(t, k_new)) return RK_ERR_SHAPE;
    vec = std::min(vec, vector_of(t));
  }
  if (!same_shape(k_new, v_new) || (q && !same_shape(q, q_out))) return RK_ERR_SHAPE;
  if (pages->k.dtype != k_new->dtype) return RK_ERR_DTYPE;
  if (pages->k.shape[1] != k_new->shape[1]) return RK_ERR_HEADS;
  if (pages->k.shape[3] != k_new->shape[rank - 1]) return RK_ERR_HEAD_DIM;
  for (const rk_tensor* t : {&pages->k, &pages->v, q_out})
    if (t && !distinct(t)) return RK_ERR_STRIDE;
  // whole requests of one length, or tokens one after the other with starts
  if (rank == 4 ? starts != nullptr || k_new->shape[0] != B : starts == nullptr && k_new->shape[0] != B)
    return RK_ERR_SHAPE;
  a.D = (int32_t)k_new->shape[rank - 1];
  const int64_t T = rank == 4 ? k_new->shape[2] : k_new->shape[0];
  if (T >= (INT64_C(1) << 31) || B >= (INT64_C(1) << 31)) return RK_ERR_SHAPE;
  const int64_t rows = rank == 4 ? B : 1;
  if (T > 0 && rows >= (INT64_C(1) << 40) / T) return RK_ERR_SHAPE;
  if (positions) {
    st = set_rotation(&a, positions, inv_freq, sections, axes, interleaved, 0, rows, T, rank == 3);
    if (st) return st;
  }
  a.T = (int32_t)T;
  a.N = rows * T;
  a.map.starts = starts;
  a.map.each = rank == 4 ? (int32_t)T : 1;
  if (q) {
    set_in(&a.part[kQ], q);
    set_out(&a.part[kQ], q_out->data, strides_of(q_out));
  }
  set_in(&a.part[kK], k_new);
  set_in(&a.part[kV], v_new);
  for (int i : {kK, kV}) {
    const rk_tensor& t = i == kK ? pages->k : pages->v;
    set_out(&a.part[i], t.data, {t.stride[0], t.stride[1], t.stride[2], t.stride[3]});
  }
  if (a.N == 0 || a.part[kQ].heads + a.part[kK].heads == 0) return RK_OK;
  if (a.part[kQ].heads && (!a.part[kQ].x || !a.part[kQ].y)) return RK_ERR_NULL;
  for (int i : {kK, kV})
    if (a.part[i].heads && (!a.part[i].x || (a.map.pages > 0 && !a.part[i].y))) return RK_ERR_NULL;
  if (B > 0 && (!a.map.lens || (cap > 0 && !a.map.table))) return RK_ERR_NULL;
  if (positions && (!a.pos || !a.freq)) return RK_ERR_NULL;
  return launch<true>(a, k_new->dtype, vec, stream);
}
