// rk_mx.hip -- quantised KV-cache rows on MI355X (gfx950): write, append and
// read back (rk_mx_write, rk_mx_append, rk_mx_read of rotatek_hip.h).
//
// Mathematics.  A block of 32 channels with largest magnitude a = m 2^x
// (m in [0.5, 1)) and an element type whose largest value is t 2^y takes
//   e = x - y + (m > t)          (t 2^y: 448 = 0.875 2^9, 6 = 0.75 2^3)
// and codes x 2^-e.  The power of two makes the product exact, so the element
// conversion is the only rounding, and code 2^e is exact in fp32.
//
// A lane holds eight channels; the four lanes of a block share its maximum by
// two lane exchanges inside the quad.  Both kernels move bytes and little
// else: 98 MB of bf16 to 51 MB of 8-bit rows takes 31 us (4.8 TB/s, the rate
// of a large copy), back 23 us (6.4 TB/s); spans of a few MB are bound by the
// launch (4 us).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "rk_common.h"
#include "rk_mx.h"

namespace {

using rk::kMxBlock;

constexpr int kThreads = 256;
constexpr int kTile = 64;  // tokens of one (batch row, head) per workgroup: a pass of 256 lanes per block of a row

struct MxArgs {
  const void* x;  // read: the output
  uint8_t* codes;
  uint8_t* scales;
  int64_t x_sb, x_sh, x_ss, x_sd;  // elements
  int64_t c_sb, c_sh, c_ss;        // bytes
  int64_t s_sb, s_sh, s_sn;
  int64_t S, cap;  // tokens in x; rows of the cache
  const int32_t* pos;
  int32_t H, D, tiles;
};

// Values pass through once, so they are loaded and stored as non-temporal and
// leave the caches to the codes, which the next kernel reads: a span of 8 x 4
// heads x 12001 tokens of 128 channels written and read back takes 54.3 us,
// 58.5 without; 32 x 8 heads x 256 tokens read back, K and V, 14.1 and 20.0.
template <class V>
__device__ __forceinline__ V load_once(const void* p) {
  return __builtin_nontemporal_load((const V*)p);
}
template <class V>
__device__ __forceinline__ void store_once(void* p, V v) {
  __builtin_nontemporal_store(v, (V*)p);
}

// Eight elements at p (stride sd), channels past nv zero.
template <class DT, bool VEC>
__device__ __forceinline__ void load_x8(const void* base, int64_t off, int64_t sd, int nv, float (&x)[8]) {
  if constexpr (DT::kBytes == 4) {
    const float* p = (const float*)base + off;
    if constexpr (VEC) {
      const rk::f32x4 a = load_once<rk::f32x4>(p), b = load_once<rk::f32x4>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < nv ? p[i * sd] : 0.f;
    }
  } else {
    uint4 w;
    if constexpr (VEC) {
      const rk::u32x4 v = load_once<rk::u32x4>((const uint16_t*)base + off);
      w = make_uint4(v[0], v[1], v[2], v[3]);
    } else {
      w = rk::load8<false>((const uint16_t*)base + off, sd, nv);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = DT::to_f32((uint16_t)(rk::word(w, i >> 1) >> (16 * (i & 1))));
  }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));  // lanes ^ 1
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));  // lanes ^ 2
}

// The block exponent byte of four lanes' eight values, and their codes.
// Magnitudes compare as their bits; an infinity or a NaN has the top
// exponent.
template <int FMT>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint2& codes) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
  a = quad_max(a);
  constexpr float kTop = FMT == RK_ROWS_MX8 ? 0.875f : 0.75f;
  constexpr int kShift = FMT == RK_ROWS_MX8 ? 9 : 3;
  const float amax = __builtin_bit_cast(float, a);
  int e = __builtin_amdgcn_frexp_expf(amax) - kShift + (__builtin_amdgcn_frexp_mantf(amax) > kTop ? 1 : 0);
  e = a == 0 ? -127 : min(max(e, -127), 127);
  const bool bad = a >= 0x7f800000u;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = bad ? 0.f : __builtin_amdgcn_ldexpf(x[i], -e);
  if constexpr (FMT == RK_ROWS_MX8) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    codes = make_uint2((uint32_t)lo, (uint32_t)hi);
  } else {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.f, 3);
    codes = make_uint2(w, 0u);
  }
  return bad ? 255u : (uint32_t)(e + 127);
}

// Write: a workgroup takes kTile tokens of one head; NB blocks a row are 4 NB
// lanes, so it holds NB passes of its 256 lanes, all loaded before the first
// is quantised.  Scales are staged in LDS and stored as runs of tokens (they
// are block-major in memory).  With `pos` rows move by the batch row's length
// and end at the capacity.
template <class DT, int FMT, int NB, bool VEC>
__device__ __forceinline__ void write_tile(const MxArgs& a, uint8_t* s_sc) {
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x / a.tiles;
  const int64_t t0 = (int64_t)(blockIdx.x % a.tiles) * kTile;
  const int64_t b = bh / a.H, h = bh - b * a.H;
  const int64_t at = a.pos ? (int64_t)max(a.pos[b], 0) : 0;
  const int64_t n = min(min(a.S, a.cap - at) - t0, (int64_t)kTile);  // tokens to write, may be <= 0
  const int64_t xo = b * a.x_sb + h * a.x_sh;
  float x[NB][8];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int f = i * kThreads + tid, t = f / (4 * NB), c = 8 * (f - t * (4 * NB));
    const int nv = t < n ? min(a.D - c, 8) : 0;
    if (nv > 0) {
      load_x8<DT, VEC>(a.x, xo + (t0 + t) * a.x_ss + c * a.x_sd, a.x_sd, nv, x[i]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[i][k] = 0.f;
    }
  }
  uint8_t* codes = a.codes + b * a.c_sb + h * a.c_sh + (at + t0) * a.c_ss;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int f = i * kThreads + tid, t = f / (4 * NB), c8 = f - t * (4 * NB);
    uint2 w;
    const uint32_t e = quantise8<FMT>(x[i], w);
    if (t < n) {
      if constexpr (FMT == RK_ROWS_MX8)
        *(uint2*)(codes + t * a.c_ss + 8 * c8) = w;
      else
        *(uint32_t*)(codes + t * a.c_ss + 4 * c8) = w.x;
    }
    if ((c8 & 3) == 0) s_sc[(c8 >> 2) * kTile + t] = (uint8_t)e;
  }
  __syncthreads();
  uint8_t* scales = a.scales + b * a.s_sb + h * a.s_sh + at + t0;
  for (int i = tid; i < NB * kTile; i += kThreads) {
    const int t = i & (kTile - 1);
    if (t < n) scales[(i / kTile) * a.s_sn + t] = s_sc[i];
  }
}

template <class DT, int FMT, int NB, bool VEC>
__global__ void __launch_bounds__(kThreads) mx_write_kernel(const MxArgs a) {
  __shared__ uint8_t s_sc[NB * kTile];
  write_tile<DT, FMT, NB, VEC>(a, s_sc);
}

// K and V of an append in one launch (blockIdx.y) where their rows hold as
// many blocks; others take a launch each.
template <class DT, int FMT, int NB, bool VEC>
__global__ void __launch_bounds__(kThreads) mx_append_kernel(const MxArgs k, const MxArgs v) {
  __shared__ uint8_t s_sc[NB * kTile];
  if (blockIdx.y == 0)
    write_tile<DT, FMT, NB, VEC>(k, s_sc);
  else
    write_tile<DT, FMT, NB, VEC>(v, s_sc);
}

// Lengths after an append, in a launch of its own: every workgroup of the
// append reads the old ones.
__global__ void __launch_bounds__(kThreads) mx_advance_kernel(int32_t* lens, int64_t B, int64_t T, int64_t cap) {
  const int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (b >= B) return;
  const int64_t n = max(lens[b], 0) + T;
  lens[b] = (int32_t)(n < cap ? n : cap);
}

// Eight channels as they are stored: code 2^e in fp32 (exact).
template <int FMT>
__device__ __forceinline__ void values8(const uint2& w, uint32_t byte, float (&y)[8]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  f2 p[4];
  if constexpr (FMT == RK_ROWS_MX8) {
    p[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false);
    p[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
    p[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false);
    p[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.f, 3);
  }
  const int e = (int)byte - 127;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = byte == 255u ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(p[i >> 1][i & 1], e);
}

template <class DT, int FMT, int NB, bool VEC>
__global__ void __launch_bounds__(kThreads) mx_read_kernel(const MxArgs a) {
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x / a.tiles;
  const int64_t t0 = (int64_t)(blockIdx.x % a.tiles) * kTile;
  const int64_t b = bh / a.H, h = bh - b * a.H;
  const int64_t n = min(a.S - t0, (int64_t)kTile);
  const uint8_t* codes = a.codes + b * a.c_sb + h * a.c_sh + t0 * a.c_ss;
  const uint8_t* scales = a.scales + b * a.s_sb + h * a.s_sh + t0;
  const int64_t xo = b * a.x_sb + h * a.x_sh;
  uint2 w[NB];
  uint32_t e[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int f = i * kThreads + tid, t = f / (4 * NB), c8 = f - t * (4 * NB);
    w[i] = make_uint2(0u, 0u);
    e[i] = 0;
    if (t < n && 8 * c8 < a.D) {
      if constexpr (FMT == RK_ROWS_MX8)
        w[i] = *(const uint2*)(codes + t * a.c_ss + 8 * c8);
      else
        w[i].x = *(const uint32_t*)(codes + t * a.c_ss + 4 * c8);
      e[i] = scales[(c8 >> 2) * a.s_sn + t];
    }
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int f = i * kThreads + tid, t = f / (4 * NB), c8 = f - t * (4 * NB);
    const int nv = t < n ? min(a.D - 8 * c8, 8) : 0;
    if (nv <= 0) continue;
    float y[8];
    values8<FMT>(w[i], e[i], y);
    const int64_t off = xo + (t0 + t) * a.x_ss + 8 * c8 * a.x_sd;
    if constexpr (DT::kBytes == 4) {
      float* p = (float*)a.x + off;
      if constexpr (VEC) {
        store_once(p, rk::f32x4{y[0], y[1], y[2], y[3]});
        store_once(p + 4, rk::f32x4{y[4], y[5], y[6], y[7]});
      } else {
        for (int k = 0; k < nv; ++k) p[k * a.x_sd] = y[k];
      }
    } else {
      uint16_t* p = (uint16_t*)a.x + off;
      if constexpr (VEC) {
        store_once(p, rk::u32x4{DT::pack2(y[0], y[1]), DT::pack2(y[2], y[3]), DT::pack2(y[4], y[5]),
                                 DT::pack2(y[6], y[7])});
      } else {
        for (int k = 0; k < nv; ++k) p[k * a.x_sd] = DT::from_f32(y[k]);
      }
    }
  }
}

// ------------------------------------------------------------------- host

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whole groups of eight channels in 16-byte pieces.
bool vec8_ok(const rk_tensor* x) {
  if (x->shape[3] % 8 != 0 || (x->stride[3] != 1 && x->shape[3] > 1)) return false;
  const int64_t align = x->dtype == RK_F32 ? 4 : 8;
  for (int i = 0; i < 3; ++i)
    if (x->shape[i] > 1 && x->stride[i] % align != 0) return false;
  return ((uintptr_t)x->data & 15) == 0;
}

// x (values) against rows: dtypes, ranks, sizes.  `T_free`: x may hold another
// number of tokens than the rows.
int check_pair(const rk_tensor* x, const rk_rows* r, bool T_free) {
  if (!x || !r) return RK_ERR_NULL;
  int st = rk::check_desc(x, 4);
  if (st) return st;
  if ((st = rk::check_mx(r))) return st;
  if (!rk::is_float_param(x->dtype)) return RK_ERR_DTYPE;
  if (x->shape[3] < 1 || x->shape[3] > 128) return RK_ERR_HEAD_DIM;
  if (x->shape[3] != r->head_dim || x->shape[0] != r->data.shape[0] || x->shape[1] != r->data.shape[1])
    return RK_ERR_SHAPE;
  if (!T_free && x->shape[2] != r->data.shape[2]) return RK_ERR_SHAPE;
  if (rk::numel(x) > 0 && !x->data) return RK_ERR_NULL;
  if (rk::numel(&r->data) > 0 && (!r->data.data || !r->scales.data)) return RK_ERR_NULL;
  return RK_OK;
}

MxArgs make_args(const rk_tensor* x, const rk_rows* r) {
  MxArgs a;
  a.x = x->data;
  a.codes = (uint8_t*)r->data.data;
  a.scales = (uint8_t*)r->scales.data;
  a.x_sb = x->stride[0]; a.x_sh = x->stride[1]; a.x_ss = x->stride[2]; a.x_sd = x->stride[3];
  a.c_sb = r->data.stride[0]; a.c_sh = r->data.stride[1]; a.c_ss = r->data.stride[2];
  a.s_sb = r->scales.stride[0]; a.s_sh = r->scales.stride[1]; a.s_sn = r->scales.stride[2];
  a.S = x->shape[2];
  a.cap = r->data.shape[2];
  a.pos = nullptr;
  a.H = (int32_t)x->shape[1];
  a.D = (int32_t)x->shape[3];
  a.tiles = (int32_t)cdiv(a.S, kTile);
  return a;
}

// f(dtype tag, format, blocks, 16-byte rows) for a call's types.
template <class F>
int by_type(int dtype, int format, int64_t nb, bool vec, F f) {
  auto blocks = [&](auto dt, auto fmt, auto v) {
    switch (nb) {
      case 1: f(dt, fmt, std::integral_constant<int, 1>{}, v); return RK_OK;
      case 2: f(dt, fmt, std::integral_constant<int, 2>{}, v); return RK_OK;
      case 3: f(dt, fmt, std::integral_constant<int, 3>{}, v); return RK_OK;
      case 4: f(dt, fmt, std::integral_constant<int, 4>{}, v); return RK_OK;
      default: return RK_ERR_HEAD_DIM;
    }
  };
  auto vecs = [&](auto dt, auto fmt) {
    return vec ? blocks(dt, fmt, std::true_type{}) : blocks(dt, fmt, std::false_type{});
  };
  auto formats = [&](auto dt) {
    return format == RK_ROWS_MX8 ? vecs(dt, std::integral_constant<int, RK_ROWS_MX8>{})
                                 : vecs(dt, std::integral_constant<int, RK_ROWS_MX4>{});
  };
  switch (dtype) {
    case RK_F16: return formats(rk::F16{});
    case RK_BF16: return formats(rk::BF16{});
    default: return formats(rk::F32{});
  }
}

int done(int st) {
  if (st) return st;
  return hipGetLastError() == hipSuccess ? RK_OK : RK_ERR_HIP;
}

// A launch has less than 2^32 threads (an append twice as many).
bool grid_ok(const MxArgs& a, int64_t B) {
  return a.S < (INT64_C(1) << 30) && B < (INT64_C(1) << 23) && B * a.H < (INT64_C(1) << 23) &&
         B * a.H * a.tiles < (INT64_C(1) << 23);
}

// Two rows at one address would be written by two workgroups at once.
bool distinct(const rk_tensor& t) {
  for (int i = 0; i < t.ndim; ++i)
    if (t.shape[i] > 1 && t.stride[i] == 0) return false;
  return true;
}

}  // namespace

extern "C" int rk_mx_write(const rk_tensor* x, const rk_rows* rows, void* stream) {
  int st = check_pair(x, rows, false);
  if (st) return st;
  if (rk::numel(x) == 0) return RK_OK;
  const MxArgs a = make_args(x, rows);
  if (!grid_ok(a, x->shape[0])) return RK_ERR_SHAPE;
  if (!distinct(rows->data) || !distinct(rows->scales)) return RK_ERR_STRIDE;
  const dim3 grid((unsigned)(x->shape[0] * a.H * a.tiles));
  st = by_type(x->dtype, rows->format, cdiv(a.D, kMxBlock), vec8_ok(x), [&](auto dt, auto fmt, auto nb, auto vec) {
    hipLaunchKernelGGL((mx_write_kernel<decltype(dt), decltype(fmt)::value, decltype(nb)::value, decltype(vec)::value>),
                       grid, dim3(kThreads), 0, (hipStream_t)stream, a);
  });
  return done(st);
}

extern "C" int rk_mx_read(const rk_rows* rows, const rk_tensor* out, void* stream) {
  int st = check_pair(out, rows, false);
  if (st) return st;
  if (rk::numel(out) == 0) return RK_OK;
  const MxArgs a = make_args(out, rows);
  if (!grid_ok(a, out->shape[0])) return RK_ERR_SHAPE;
  if (!distinct(*out)) return RK_ERR_STRIDE;
  const dim3 grid((unsigned)(out->shape[0] * a.H * a.tiles));
  st = by_type(out->dtype, rows->format, cdiv(a.D, kMxBlock), vec8_ok(out), [&](auto dt, auto fmt, auto nb, auto vec) {
    hipLaunchKernelGGL((mx_read_kernel<decltype(dt), decltype(fmt)::value, decltype(nb)::value, decltype(vec)::value>),
                       grid, dim3(kThreads), 0, (hipStream_t)stream, a);
  });
  return done(st);
}

extern "C" int rk_mx_append(const rk_tensor* k_new, const rk_tensor* v_new, const rk_rows* k_rows,
                            const rk_rows* v_rows, int32_t* lens, int32_t advance, void* stream) {
  int st = check_pair(k_new, k_rows, true);
  if (st) return st;
  if ((v_new == nullptr) != (v_rows == nullptr)) return RK_ERR_NULL;
  if (v_new) {
    if ((st = check_pair(v_new, v_rows, true))) return st;
    for (int i = 0; i < 3; ++i)
      if (k_new->shape[i] != v_new->shape[i]) return RK_ERR_SHAPE;
    if (k_rows->data.shape[2] != v_rows->data.shape[2]) return RK_ERR_SHAPE;
    if (k_new->dtype != v_new->dtype || k_rows->format != v_rows->format) return RK_ERR_DTYPE;
  }
  const int64_t B = k_new->shape[0], T = k_new->shape[2], cap = k_rows->data.shape[2];
  if (B == 0) return RK_OK;
  if (!lens) return RK_ERR_NULL;
  if (T == 0 || k_new->shape[1] == 0) return RK_OK;
  if (cap >= (INT64_C(1) << 31)) return RK_ERR_SHAPE;
  MxArgs k = make_args(k_new, k_rows), v = v_new ? make_args(v_new, v_rows) : k;
  if (!grid_ok(k, B)) return RK_ERR_SHAPE;
  for (const rk_rows* r : {k_rows, v_rows})
    if (r && (!distinct(r->data) || !distinct(r->scales))) return RK_ERR_STRIDE;
  k.pos = v.pos = lens;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(B * k.H * k.tiles));
  if (cap > 0) {
    const int64_t nbk = cdiv(k.D, kMxBlock), nbv = cdiv(v.D, kMxBlock);
    const bool vec = vec8_ok(k_new) && (!v_new || vec8_ok(v_new));
    if (v_new && nbk == nbv) {
      st = by_type(k_new->dtype, k_rows->format, nbk, vec, [&](auto dt, auto fmt, auto nb, auto vc) {
        constexpr int NB = decltype(nb)::value;
        hipLaunchKernelGGL((mx_append_kernel<decltype(dt), decltype(fmt)::value, NB, decltype(vc)::value>),
                           dim3(grid.x, 2), dim3(kThreads), 0, s, k, v);
      });
    } else {
      for (int i = 0; i < (v_new ? 2 : 1) && !st; ++i) {
        const MxArgs a = i ? v : k;
        st = by_type(k_new->dtype, k_rows->format, i ? nbv : nbk, vec, [&](auto dt, auto fmt, auto nb, auto vc) {
          constexpr int NB = decltype(nb)::value;
          hipLaunchKernelGGL((mx_write_kernel<decltype(dt), decltype(fmt)::value, NB, decltype(vc)::value>), grid,
                             dim3(kThreads), 0, s, a);
        });
      }
    }
  }
  if (st == RK_OK && advance)
    hipLaunchKernelGGL(mx_advance_kernel, dim3((unsigned)cdiv(B, kThreads)), dim3(kThreads), 0, s, lens, B, T, cap);
  return done(st);
}
