// rk_span_mx8.hip -- span attention over quantised rows of 8-bit codes
// (kernels in rk_span_dev.h).
#include "rk_span_dev.h"

namespace rk {

using F = Mx8Fmt;

// terms 2: bf16 and fp16 queries, exact in two bf16 terms, probabilities in
// two; 3: fp32 ones, exact in three, probabilities in three.
hipError_t span_launch_mx8(int kv, int kf, int terms, const SpanArgs& a, unsigned grid, hipStream_t s) {
  return terms == 3 ? pick_widths<F, 3, 3, true>(kv, kf, a, grid, s) : pick_widths<F, 2, 2, true>(kv, kf, a, grid, s);
}

hipError_t span_join_mx8(int kf, const SpanArgs& a, unsigned grid, hipStream_t s) {
  return pick_join<F, 2, 2>(kf, a, grid, s);
}

}  // namespace rk
