// The few-rows kernel over 8-bit keys and 8-bit values.
#include "tq_affine_rows.h"

namespace tq {

int launch_rows_k8v8(const AffineAttnParams& p, const RowsChoice& r, int dtype, hipStream_t st) {
  return dtype == TQ_DTYPE_F16 ? launch_rows_bits<TQ_DTYPE_F16, 8, 8>(p, r, st)
                               : launch_rows_bits<TQ_DTYPE_BF16, 8, 8>(p, r, st);
}

}  // namespace tq
