// The many-rows kernel over 4-bit keys and 4-bit values.
#include "tq_affine_tile.h"

namespace tq {

int launch_tile_k4v4(const AffineAttnParams& p, int dtype, hipStream_t st) {
  return dtype == TQ_DTYPE_F16 ? launch_tile_bits<TQ_DTYPE_F16, 4, 4>(p, st)
                               : launch_tile_bits<TQ_DTYPE_BF16, 4, 4>(p, st);
}

}  // namespace tq
