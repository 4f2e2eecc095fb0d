// rk_tile_mx4.hip -- attention over shared rows of this format (kernels in
// rk_tile_dev.h): terms of a query, and of a probability, as in rk_span_mx4.hip.
#include "rk_tile_dev.h"

namespace rk {

hipError_t tile_launch_mx4(int kv, int kf, const SpanArgs& a, unsigned grid, hipStream_t s) {
  return pick_tiles<Mx4Fmt, 2, 2>(kv, kf, a, grid, s);
}

}  // namespace rk
