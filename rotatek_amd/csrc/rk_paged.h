// rk_paged.h -- the argument block of the attention over pages or plain rows
// that its host code (rk_paged.hip) and kernels share, and the checks of a pool
// of pages.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rk_host.h"
#include "rk_page_map.h"

namespace rk {

// Workgroups of 256 threads that a launch has less than: its threads are counted in
// 32 bits.
constexpr int64_t kMostGroups = INT64_C(1) << 24;

// Checks a pool and its table; *B requests, *cap tokens each at most.
inline int set_pages(const rk_pages* p, PageMap* m, int64_t* B, int64_t* cap) {
  int st;
  if ((st = check_desc(&p->k, 4)) || (st = check_desc(&p->v, 4)) || (st = check_desc(&p->table, 2))) return st;
  if (!is_float_param(p->k.dtype) || p->v.dtype != p->k.dtype || p->table.dtype != RK_I32) return RK_ERR_DTYPE;
  for (int i = 0; i < 4; ++i)
    if (p->k.shape[i] != p->v.shape[i]) return RK_ERR_SHAPE;
  const int64_t page = p->k.shape[2];
  if (page < kMinPage || (page & (page - 1)) || page > (1 << 20)) return RK_ERR_SHAPE;
  if (p->k.shape[0] >= (INT64_C(1) << 31) || p->table.shape[0] >= (INT64_C(1) << 31)) return RK_ERR_SHAPE;
  if (p->table.shape[1] > ((INT64_C(1) << 31) - page) / page) return RK_ERR_SHAPE;
  if (p->table.stride[1] != 1 && p->table.shape[1] > 1) return RK_ERR_STRIDE;
  if (p->k.shape[3] < 1 || p->k.shape[3] > 128) return RK_ERR_HEAD_DIM;
  int shift = 0;
  while ((INT64_C(1) << shift) < page) ++shift;
  m->table = (const int32_t*)p->table.data;
  m->lens = p->lens;
  m->t_sb = p->table.stride[0];
  m->B = (int32_t)p->table.shape[0];
  m->per = (int32_t)p->table.shape[1];
  m->pages = (int32_t)p->k.shape[0];
  m->shift = shift;
  *B = m->B;
  *cap = p->table.shape[1] * page;
  m->cap = (int32_t)*cap;
  return RK_OK;
}

struct PagedArgs {
  PageMap map;
  const void *q, *k, *v;
  void* out;
  // elements; q and out of token n of request b: n (starts) or b, n
  int64_t q_sb, q_st, q_sh, q_sd, o_sb, o_st, o_sh, o_sd;
  int64_t k_sp, k_sh, k_ss, v_sp, v_sh, v_ss;
  float *acc, *ml;  // partial records
  int2* span;       // one new token each: first and last share of a unit
  int64_t N;        // new tokens in all
  int32_t Hq, H, G, D, T;  // T: new tokens of each request (0: starts)
  int32_t window, sinks;   // window INT_MAX: none
  int32_t workers;         // one new token each: workgroups of the split launch
  int32_t direct;          // ... waves of one that takes a unit by itself (0: shares and a join)
  int32_t splits;          // many: parts that a row's tokens are cut into
  int32_t round;           // ... workgroups of a KV head that CUs take one each of, where all begin at once (0: not)
  int32_t q_vec, o_vec;
  float scale_log2;  // log2(e) / sqrt(D)
};

// The launches over many new tokens a request (rk_window.hip); a status.
// Slots: workgroups of a KV head and split.
int64_t window_slots(const PagedArgs& a);
int window_per_cu(const PagedArgs& a);  // workgroups that a CU holds
int window_launch(const PagedArgs& a, int32_t dtype, hipStream_t s);

}  // namespace rk
