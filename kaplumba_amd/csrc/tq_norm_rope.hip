// Norms of the queries and keys of each head and the rotation by their positions, in one pass.
#include "tq_common.h"

namespace tq {
namespace {

constexpr int kMaxDim = 512;
constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)

struct NormRopeParams {
  const void* x[2];  // queries, keys
  int64_t sb[2], sh[2], sl[2];
  const void* w[2];
  void* out[2];
  int H[2];
  int B, L, dim, rot;
  int adjacent, weight_dtype;
  float eps, factor;
  const float* inv_freq;
  const int32_t* axis;
  int axes;
  const void* pos;
  int pos_wide;  // 64-bit positions
  int64_t pos_start, pos_sa, pos_sb, pos_sl;
  int64_t rows;  // B * L * (Hq + Hk)
};

__device__ __forceinline__ int64_t position(const NormRopeParams& p, int a, int b, int l) {
  if (!p.pos) return p.pos_start + l;
  const int64_t at = a * p.pos_sa + b * p.pos_sb + l * p.pos_sl;
  return p.pos_wide ? static_cast<const int64_t*>(p.pos)[at] : static_cast<const int32_t*>(p.pos)[at];
}

// cos and sin of pos * inv_freq times the factor.  The angle is taken in turns in 64 bits, where a position of a
// million loses 2^-30 of a turn at most; 32 bits would be off by whole percents of a radian there.  The rest of
// less than half a turn goes into 32 bits.
__device__ __forceinline__ float2 turn(const NormRopeParams& p, int i, int b, int l) {
  const int a = p.axis ? min(max(p.axis[i], 0), p.axes - 1) : 0;
  const double t = static_cast<double>(position(p, a, b, l)) * (static_cast<double>(p.inv_freq[i]) * kTurn);
  float s, c;
  sincospif(static_cast<float>(2.0 * (t - rint(t))), &s, &c);
  return make_float2(c * p.factor, s * p.factor);
}

__device__ __forceinline__ float weight_at(const NormRopeParams& p, int side, int d) {
  return p.weight_dtype == TQ_DTYPE_F32   ? load_elem<TQ_DTYPE_F32>(p.w[side], d)
         : p.weight_dtype == TQ_DTYPE_F16 ? load_elem<TQ_DTYPE_F16>(p.w[side], d)
                                          : load_elem<TQ_DTYPE_BF16>(p.w[side], d);
}

// y = x / sqrt(mean(x^2) + eps) * w, then the pairs of the first rot coordinates turned; everything in f32,
// rounded once at the end.  One wave a row, element loads: any dim and stride.
template <int DT>
__global__ __launch_bounds__(256) void norm_rope_kernel(const NormRopeParams p) {
  __shared__ float row_y[4][kMaxDim];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t r = min(static_cast<int64_t>(blockIdx.x) * 4 + wave, p.rows - 1);
  const int heads = p.H[0] + p.H[1];
  const int64_t token = r / heads;
  int h = static_cast<int>(r - token * heads);
  const int side = h >= p.H[0];
  h -= side ? p.H[0] : 0;
  const int64_t b64 = token / p.L;
  const int b = static_cast<int>(b64), l = static_cast<int>(token - b64 * p.L);
  const int64_t from = b * p.sb[side] + h * p.sh[side] + l * p.sl[side];
  float* y = row_y[wave];
  float sum = 0.f;
  for (int d = lane; d < p.dim; d += 64) {
    const float v = load_elem<DT>(p.x[side], from + d);
    y[d] = v;
    sum = __builtin_fmaf(v, v, sum);
  }
  if (p.w[side]) {
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    const float inv = 1.f / sqrtf(sum / static_cast<float>(p.dim) + p.eps);
    for (int d = lane; d < p.dim; d += 64) y[d] = y[d] * inv * weight_at(p, side, d);
  }
  __syncthreads();
  const int64_t to = ((b64 * p.H[side] + h) * p.L + l) * p.dim;
  const int half = p.rot / 2;
  if (static_cast<int64_t>(blockIdx.x) * 4 + wave >= p.rows) return;
  for (int i = lane; i < half; i += 64) {
    const float2 cs = turn(p, i, b, l);
    const int j = p.adjacent ? 2 * i : i, k = p.adjacent ? 2 * i + 1 : i + half;
    const float u = y[j], v = y[k];
    store_elem<DT>(p.out[side], to + j, u * cs.x - v * cs.y);
    store_elem<DT>(p.out[side], to + k, u * cs.y + v * cs.x);
  }
  for (int d = p.rot + lane; d < p.dim; d += 64) store_elem<DT>(p.out[side], to + d, y[d]);
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" int tq_norm_rope(const void* q, const void* k, int dtype, int B, int Hq, int Hk, int L, int dim,
                            int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, int64_t k_stride_b,
                            int64_t k_stride_h, int64_t k_stride_l, const void* q_weight, const void* k_weight,
                            int weight_dtype, float eps, int rot_dim, int adjacent, const float* inv_freq, float factor,
                            const int32_t* axis, int axes, const void* positions, int position_bytes, int64_t start,
                            int64_t pos_stride_a, int64_t pos_stride_b, int64_t pos_stride_l, void* q_out, void* k_out,
                            void* stream) {
  const char* what = "tq_norm_rope";
  if (dtype < TQ_DTYPE_F32 || dtype > TQ_DTYPE_BF16) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: dtype %d", what, dtype);
  if (B < 0 || Hq < 0 || Hk < 0 || L < 0)
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: bad sizes B=%d, heads %d and %d, L=%d", what, B, Hq, Hk, L);
  if (dim < 2 || dim > kMaxDim) return fail(TQ_ERR_UNSUPPORTED, "%s: head dim %d (2..%d)", what, dim, kMaxDim);
  if (rot_dim < 0 || rot_dim > dim || rot_dim % 2)
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: %d rotated of %d coordinates", what, rot_dim, dim);
  if (axes < 1 || (axes > 1 && !axis)) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: %d axes without their frequencies' table", what, axes);
  if (axes > 1 && !positions) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: several axes need positions", what);
  if (positions && position_bytes != 4 && position_bytes != 8)
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: positions of %d bytes", what, position_bytes);
  if ((q_weight || k_weight) && (weight_dtype < TQ_DTYPE_F32 || weight_dtype > TQ_DTYPE_BF16))
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: weight_dtype %d", what, weight_dtype);
  if (!(eps >= 0.f)) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: eps %g", what, eps);
  if (B == 0 || L == 0 || Hq + Hk == 0) return TQ_OK;
  if ((Hq && (!q || !q_out)) || (Hk && (!k || !k_out)) || (rot_dim && !inv_freq))
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  NormRopeParams p{};
  p.x[0] = q, p.x[1] = k;
  p.sb[0] = q_stride_b, p.sh[0] = q_stride_h, p.sl[0] = q_stride_l;
  p.sb[1] = k_stride_b, p.sh[1] = k_stride_h, p.sl[1] = k_stride_l;
  p.w[0] = q_weight, p.w[1] = k_weight;
  p.out[0] = q_out, p.out[1] = k_out;
  p.H[0] = Hq, p.H[1] = Hk;
  p.B = B, p.L = L, p.dim = dim, p.rot = rot_dim;
  p.adjacent = adjacent, p.weight_dtype = weight_dtype;
  p.eps = eps, p.factor = factor;
  p.inv_freq = inv_freq, p.axis = axis, p.axes = axes;
  p.pos = positions, p.pos_wide = position_bytes == 8, p.pos_start = start;
  p.pos_sa = pos_stride_a, p.pos_sb = pos_stride_b, p.pos_sl = pos_stride_l;
  p.rows = static_cast<int64_t>(B) * L * (static_cast<int64_t>(Hq) + Hk);
  const int64_t blocks = (p.rows + 3) / 4;
  if (blocks > INT32_MAX / 256) return fail(TQ_ERR_UNSUPPORTED, "%s: %lld vectors in one call", what, static_cast<long long>(p.rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned n = static_cast<unsigned>(blocks);
  if (dtype == TQ_DTYPE_F32)
    norm_rope_kernel<TQ_DTYPE_F32><<<n, 256, 0, st>>>(p);
  else if (dtype == TQ_DTYPE_F16)
    norm_rope_kernel<TQ_DTYPE_F16><<<n, 256, 0, st>>>(p);
  else
    norm_rope_kernel<TQ_DTYPE_BF16><<<n, 256, 0, st>>>(p);
  return check_launch(what);
}
