// rk_span_f16.hip -- span attention over plain f16 rows (kernels in
// rk_span_dev.h): queries exact in one term, probabilities in two.
#include "rk_span_dev.h"

namespace rk {

using F = PlainFmt<F16>;

hipError_t span_launch_f16(int kv, int kf, bool vec, const SpanArgs& a, unsigned grid, hipStream_t s) {
  return vec ? pick_widths<F, 1, 2, true>(kv, kf, a, grid, s) : pick_widths<F, 1, 2, false>(kv, kf, a, grid, s);
}

hipError_t span_join_f16(int kf, const SpanArgs& a, unsigned grid, hipStream_t s) {
  return pick_join<F, 1, 2>(kf, a, grid, s);
}

}  // namespace rk
