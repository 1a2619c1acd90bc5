// Norms of the queries and keys of each head and the rotation by their positions, in one pass:
//   y = x / sqrt(mean(x^2) + eps) * w over the head, then pairs (y_i, y_j) -> (c y_i - s y_j, s y_i + c y_j).
// Bound by memory: each input read once and each output written once.  8192 tokens of 40 heads of 128, bf16 (168 MB): 29
// us, 5.8 TB/s (a good part of it stays in the caches between two such calls; single elements instead of pieces: 177
// us); one token: 4 us, the latency of a load, a sum and the angles.
#include <algorithm>

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
// rounded once at the end.  One wave a row, element loads: any dim and stride.  Its double-precision turns, found
// again for every head, bound it: 8192 tokens of 40 heads of 128, 180 us.
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

// Eight consecutive elements as f32 in 16-byte loads, and back.
template <int DT>
struct Eight {
  uint4 w[DT == TQ_DTYPE_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* x, int64_t at) {
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const char*>(x) + at * (DT == TQ_DTYPE_F32 ? 4 : 2));
    w[0] = from[0];
    if constexpr (DT == TQ_DTYPE_F32) w[1] = from[1];
  }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < (DT == TQ_DTYPE_F32 ? 2 : 1); ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DT == TQ_DTYPE_F32) {
          v[4 * i + j] = __uint_as_float(u[j]);
        } else if constexpr (DT == TQ_DTYPE_F16) {
          v[2 * j] = f16_bits_to_f32(u[j] & 0xffffu), v[2 * j + 1] = f16_bits_to_f32(u[j] >> 16);
        } else {
          v[2 * j] = __uint_as_float(u[j] << 16), v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
      }
    }
  }
  __device__ __forceinline__ void put(const float* v) {
    if constexpr (DT == TQ_DTYPE_F32) {
      w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DT == TQ_DTYPE_F16) {
          typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
          const half2_t t = {static_cast<_Float16>(v[2 * j]), static_cast<_Float16>(v[2 * j + 1])};
          u[j] = __builtin_bit_cast(uint32_t, t);
        } else {
          typedef __bf16 bhalf2_t __attribute__((ext_vector_type(2)));
          const bhalf2_t t = {static_cast<__bf16>(v[2 * j]), static_cast<__bf16>(v[2 * j + 1])};
          u[j] = __builtin_bit_cast(uint32_t, t);
        }
      }
      w[0] = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
  __device__ __forceinline__ void store(void* x, int64_t at) const {
    uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(x) + at * (DT == TQ_DTYPE_F32 ? 4 : 2));
    to[0] = w[0];
    if constexpr (DT == TQ_DTYPE_F32) to[1] = w[1];
  }
};

// The same for dims and rotated parts that are multiples of 16, in 16-byte pieces.  A lane holds 16 coordinates of
// one head, the eight pairs that frequencies 8 j .. 8 j + 7 turn (or 16 that are not turned: cos 1, sin 0), LH lanes
// a head (dim / 16 of them in use) and 64 / LH heads a wave at a time.  A wave takes one token: its lanes find one
// frequency's cosine and sine each, once for all heads, and hand them round through LDS; the next heads load while
// these are worked on.  Bound by memory where tokens are many; a few tokens are spread over the chip by heads.
template <int DT, int LH, bool ADJ>
__global__ __launch_bounds__(256) void norm_rope_pieces_kernel(const NormRopeParams p, int head_parts, int part_steps) {
  constexpr int HW = 64 / LH;  // heads a step
  __shared__ float2 turns[4][kMaxDim / 2];
  __shared__ float weights[2][kMaxDim];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < 2 * p.dim; i += 256) {
    const int side = i >= p.dim, d = i - (side ? p.dim : 0);
    weights[side][d] = p.w[side] ? weight_at(p, side, d) : 1.f;
  }
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;  // (token, part of the heads)
  const int64_t tokens = static_cast<int64_t>(p.B) * p.L;
  const int64_t token = min(unit / head_parts, tokens - 1);
  const int part = static_cast<int>(unit % head_parts);
  const bool live = unit < tokens * head_parts;
  const int64_t b64 = token / p.L;
  const int b = static_cast<int>(b64), l = static_cast<int>(token - b64 * p.L);

  const int heads = p.H[0] + p.H[1];
  const int j = lane % LH, in_step = lane / LH;
  const int rot_pieces = p.rot / 16, pieces = p.dim / 16;
  const bool used = j < pieces, turned = j < rot_pieces;
  const int jj = used ? j : 0;
  const int at0 = turned && !ADJ ? 8 * jj : 16 * jj;
  const int at1 = turned && !ADJ ? 8 * jj + p.rot / 2 : 16 * jj + 8;
  const int first = part * part_steps * HW;
  const int stop = min(heads, first + part_steps * HW);

  Eight<DT> in[2], next[2];
  auto load = [&](int h0, Eight<DT> (&to)[2]) {
    const int h = min(h0 + in_step, heads - 1);
    const bool key = h >= p.H[0];
    const int64_t from = b * (key ? p.sb[1] : p.sb[0]) + (h - (key ? p.H[0] : 0)) * (key ? p.sh[1] : p.sh[0]) +
                         l * (key ? p.sl[1] : p.sl[0]);
    const void* x = key ? p.x[1] : p.x[0];
    to[0].load(x, from + at0);
    to[1].load(x, from + at1);
  };
  load(first, in);
  for (int i = lane; i < p.rot / 2; i += 64) turns[wave][i] = turn(p, i, b, l);
  __syncthreads();
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 t = turned ? turns[wave][8 * jj + i] : make_float2(1.f, 0.f);
    cs[i] = t.x, sn[i] = t.y;
  }
  if (!live) return;
  const float inv_dim = 1.f / static_cast<float>(p.dim);
  for (int h0 = first; h0 < stop; h0 += HW) {
    if (h0 + HW < stop) load(h0 + HW, next);
    const int h = min(h0 + in_step, heads - 1);
    const bool key = h >= p.H[0];
    float v[16];
    in[0].get(v);
    in[1].get(v + 8);
    if (key ? p.w[1] : p.w[0]) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(v[i], v[i], sum);
      sum = used ? sum : 0.f;
      if constexpr (LH >= 2) sum += xor_lane<1>(sum);
      if constexpr (LH >= 4) sum += xor_lane<2>(sum);
      if constexpr (LH >= 8) sum += xor_lane<4>(sum);
      if constexpr (LH >= 16) sum += xor_lane<8>(sum);
      if constexpr (LH >= 32) sum += xor_lane<16>(sum);
      const float inv = 1.f / sqrtf(__builtin_fmaf(sum, inv_dim, p.eps));
      const float* w = weights[key];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = v[i] * inv * w[at0 + i];
        v[8 + i] = v[8 + i] * inv * w[at1 + i];
      }
    }
    float o[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int a = ADJ ? 2 * i : i, c = ADJ ? 2 * i + 1 : i + 8;
      o[a] = v[a] * cs[i] - v[c] * sn[i];
      o[c] = v[a] * sn[i] + v[c] * cs[i];
    }
    // what is not turned stays as it is, an infinity too
    if (!turned) {
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = v[i];
    }
    if (used && h0 + in_step < stop) {
      const int64_t to = ((b64 * (key ? p.H[1] : p.H[0]) + (h - (key ? p.H[0] : 0))) * p.L + l) * p.dim;
      void* out = key ? p.out[1] : p.out[0];
      Eight<DT> r;
      r.put(o);
      r.store(out, to + at0);
      r.put(o + 8);
      r.store(out, to + at1);
    }
    in[0] = next[0], in[1] = next[1];
  }
}

bool aligned16(const void* x, int64_t a, int64_t b, int64_t c, int item) {
  return ((reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>((a | b | c) * item)) & 15) == 0;
}

template <int DT, int LH>
void launch_pieces(const NormRopeParams& p, hipStream_t st) {
  constexpr int HW = 64 / LH;
  const int steps = (p.H[0] + p.H[1] + HW - 1) / HW;
  const int64_t tokens = static_cast<int64_t>(p.B) * p.L;
  // Enough waves for two on every SIMD before one takes several steps of heads, for which the angles are worked out
  // once (1024 tokens: 8.6 us, 9.7 with half a wave a SIMD, 8.3 with eight; 8192 tokens 32.2, 32.0, 32.5).
  const int64_t waves = static_cast<int64_t>(device_cu_count()) * 8;
  const int parts = static_cast<int>(std::min<int64_t>(steps, std::max<int64_t>(1, waves / tokens)));
  const int part_steps = (steps + parts - 1) / parts;
  const int used_parts = (steps + part_steps - 1) / part_steps;
  const unsigned n = static_cast<unsigned>((tokens * used_parts + 3) / 4);
  if (p.adjacent)
    norm_rope_pieces_kernel<DT, LH, true><<<n, 256, 0, st>>>(p, used_parts, part_steps);
  else
    norm_rope_pieces_kernel<DT, LH, false><<<n, 256, 0, st>>>(p, used_parts, part_steps);
}

template <int DT>
void launch(const NormRopeParams& p, bool pieces, unsigned rows4, hipStream_t st) {
  if (!pieces)
    norm_rope_kernel<DT><<<rows4, 256, 0, st>>>(p);
  else if (p.dim <= 64)
    launch_pieces<DT, 4>(p, st);
  else if (p.dim <= 128)
    launch_pieces<DT, 8>(p, st);
  else if (p.dim <= 256)
    launch_pieces<DT, 16>(p, st);
  else
    launch_pieces<DT, 32>(p, st);
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
  // 16-byte pieces where every row has them, single elements elsewhere (8192 tokens 29 us / 177 us, one token 4 / 5)
  const int item = dtype == TQ_DTYPE_F32 ? 4 : 2;
  const bool pieces = dim % 16 == 0 && rot_dim % 16 == 0 && (!Hq || aligned16(q, q_stride_b, q_stride_h, q_stride_l, item)) &&
                      (!Hk || aligned16(k, k_stride_b, k_stride_h, k_stride_l, item)) && aligned16(q_out, 0, 0, 0, item) &&
                      aligned16(k_out, 0, 0, 0, item);
  if (dtype == TQ_DTYPE_F32)
    launch<TQ_DTYPE_F32>(p, pieces, n, st);
  else if (dtype == TQ_DTYPE_F16)
    launch<TQ_DTYPE_F16>(p, pieces, n, st);
  else
    launch<TQ_DTYPE_BF16>(p, pieces, n, st);
  return check_launch(what);
}
