// The few-rows kernel over 4-bit keys and 4-bit values.
#include "tq_affine_rows.h"

namespace tq {

int launch_rows_k4v4(const AffineAttnParams& p, const RowsChoice& r, int dtype, hipStream_t st) {
  return dtype == TQ_DTYPE_F16 ? launch_rows_bits<TQ_DTYPE_F16, 4, 4>(p, r, st)
                               : launch_rows_bits<TQ_DTYPE_BF16, 4, 4>(p, r, st);
}

}  // namespace tq
