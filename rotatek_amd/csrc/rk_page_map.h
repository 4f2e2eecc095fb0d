// rk_page_map.h -- where the tokens of a paged KV cache lie.
//
// Lengths, starts and page numbers come from device memory; every one is
// checked here before it becomes an address.  A length counts as far as the
// table reaches, and a token whose page is not in the pool is not there.  No HIP
// in here but the attributes: the same code runs on the host for its tests.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define RK_EVERYWHERE __host__ __device__ __forceinline__
#else
#define RK_EVERYWHERE inline
#endif

namespace rk {

constexpr int kMinPage = 8;  // rows: eight neighbouring tokens, as the kernels read them, lie in one page

struct PageMap {
  const int32_t* table;   // [B, per], or null: request b's one page is b (plain rows)
  const int32_t* lens;    // [B], or null: every request fills its table
  const int32_t* starts;  // [B + 1], or null: `each` new tokens a request
  int64_t t_sb;           // elements from a request's table to the next
  int32_t B, per, pages, each;
  int32_t shift, cap;  // log2 rows of a page; tokens that a table reaches
};

// Tokens that request b holds.
RK_EVERYWHERE int len_of(const PageMap& m, int b) {
  if (!m.lens) return m.cap;
  const int n = m.lens[b];
  return n < 0 ? 0 : n > m.cap ? m.cap : n;
}

// The page of token j (below cap) of request b; outside the pool: none.
RK_EVERYWHERE uint32_t page_of(const PageMap& m, int b, int j) {
  return m.table ? (uint32_t)m.table[b * m.t_sb + (j >> m.shift)] : (uint32_t)b;
}

// The last request whose first new token is at or before n (starts ascend).
RK_EVERYWHERE int request_of(const int32_t* starts, int B, int64_t n) {
  int low = 0, high = B;  // starts[low] <= n < starts[high], if it is anywhere
  while (high - low > 1) {
    const int mid = (int)(((int64_t)low + high) >> 1);
    if (starts[mid] <= n) low = mid; else high = mid;
  }
  return low;
}

// Page and row that new token n of request b's s .. e - 1 goes to, which holds `len`
// with them; a negative page where it goes nowhere.
RK_EVERYWHERE int64_t place_in(const PageMap& m, int64_t n, int64_t b, int64_t s, int64_t e, int64_t len, int* row) {
  const int64_t p = len - e + n;
  if (n < s || n >= e || p < 0 || p >= m.cap) return -1;
  const uint32_t page = page_of(m, (int)b, (int)p);
  if (page >= (uint32_t)m.pages) return -1;
  *row = (int)p & ((1 << m.shift) - 1);
  return page;
}

// The same, b: request_of n (where there are starts).
RK_EVERYWHERE int64_t place_of(const PageMap& m, int64_t n, int64_t b, int* row) {
  if (m.B <= 0) return -1;
  int64_t s, e;  // the request's new tokens
  if (m.starts) {
    s = m.starts[b];
    e = m.starts[b + 1];
  } else {
    b = n / m.each;
    s = b * m.each;
    e = s + m.each;
  }
  return place_in(m, n, b, s, e, m.lens[b], row);
}

// The tokens that queries at positions lo_p .. hi_p (lo_p from 0 on) see, as
// blocks of W tokens that start at multiples of W: the sinks' first, then the
// window's.
template <int W>
struct Seen {
  int low;     // first token of the window's first block
  int sinks;   // blocks of sinks ahead of it
  int blocks;  // in all
  RK_EVERYWHERE Seen(int lo_p, int hi_p, int window, int n_sinks) {
    const int first = lo_p - window + 1;
    low = first < 0 ? 0 : first & ~(W - 1);
    sinks = ((n_sinks < low ? n_sinks : low) + W - 1) / W;
    blocks = hi_p < 0 ? 0 : sinks + (hi_p - low) / W + 1;
    if (sinks > blocks) sinks = blocks;
  }
  RK_EVERYWHERE int token(int i) const { return i < sinks ? i * W : low + (i - sinks) * W; }
};

// Whether the query at position p sees token j.
RK_EVERYWHERE bool sees(int p, int j, int window, int sinks) { return j <= p && (p - j < window || j < sinks); }

}  // namespace rk
