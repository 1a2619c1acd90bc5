// The many-rows kernel over 8-bit keys and 8-bit values.
#include "tq_affine_tile.h"

namespace tq {

int launch_tile_k8v8(const AffineAttnParams& p, int dtype, hipStream_t st) {
  return dtype == TQ_DTYPE_F16 ? launch_tile_bits<TQ_DTYPE_F16, 8, 8>(p, st)
                               : launch_tile_bits<TQ_DTYPE_BF16, 8, 8>(p, st);
}

}  // namespace tq
