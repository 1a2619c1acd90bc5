// The group-affine cache's write and read back.
#include "tq_affine.h"

namespace tq {
namespace {

// One side (keys or values) of an append.
struct AffineSide {
  const void* x;
  int64_t sb, sh, sl;
  uint32_t* codes;
  void* params;
  int dim, bits;
  int64_t chunks;  // B * H * L * dim / 8
};

struct AffineAppendParams {
  AffineSide side[2];
  int64_t k_blocks;  // workgroups of the keys; the rest are the values'
  int H, L, group;
  int64_t capacity, offset;
};

// Eight consecutive elements of x as f32, in 16-byte loads where the host found them aligned.
template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t at, float (&v)[8]) {
  if constexpr (DT == TQ_DTYPE_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(x) + at + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == TQ_DTYPE_F16) {
        v[2 * i] = f16_bits_to_f32(w[i] & 0xffffu);
        v[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ void store_pair(void* params, int64_t i, float s, float b) {
  if constexpr (DT == TQ_DTYPE_F32)
    static_cast<float2*>(params)[i] = make_float2(s, b);
  else if constexpr (DT == TQ_DTYPE_F16)
    static_cast<uint32_t*>(params)[i] = f32_to_f16_bits(s) | static_cast<uint32_t>(f32_to_f16_bits(b)) << 16;
  else
    static_cast<uint32_t*>(params)[i] = f32_to_bf16_bits(s) | static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16;
}

template <int OFF>
__device__ __forceinline__ void range_step(float& lo, float& hi, uint32_t& top) {
  lo = fminf(lo, xor_lane<OFF>(lo));
  hi = fmaxf(hi, xor_lane<OFF>(hi));
  top = max(top, __float_as_uint(xor_lane<OFF>(__uint_as_float(top))));
}

// A lane holds eight coordinates of one row, group / 8 neighbouring lanes a group:
//   lo, hi = the group's least and greatest value, s = T((hi - lo) / n), n = 2^bits - 1, bias = lo,
//   code = the number of half steps (k + 1/2) s, k = 0 .. n - 1, that d = x - lo (in f32) reaches.
// Differences are taken in halves, so that they stay finite.  d / s lies within an ulp of d * (1 / s); the residual
// d - k s is exact in an fma (both are multiples of ulp(s) and it is at most s), which settles the border.
// Scales below 2^-100 count as 0 (every code 0), so that 1 / s and the halves stay normal.
// s and bias are of the vectors' own type: lo is then exact, and s off by half a step at most over the whole
// range (2^-9 of it in bf16, 1/255 of it is a step at 8 bits).  A group with a value that is not finite gets NaN
// for both, and codes of 0.
template <int DT, int BITS>
__device__ __forceinline__ void append_chunk(const AffineAppendParams& p, const AffineSide& s, int64_t i, bool live) {
  const int per_row = s.dim >> 3;
  const int64_t row = i / per_row;
  const int c = static_cast<int>(i - row * per_row);
  const int64_t bh = row / p.L;
  const int l = static_cast<int>(row - bh * p.L);
  const int64_t b = bh / p.H;
  const int h = static_cast<int>(bh - b * p.H);
  float v[8];
  load8<DT>(s.x, b * s.sb + h * s.sh + l * s.sl + c * 8, v);
  float lo = v[0], hi = v[0];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo = fminf(lo, v[j]);
    hi = fmaxf(hi, v[j]);
    top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  }
  range_step<1>(lo, hi, top);
  range_step<2>(lo, hi, top);
  if (p.group >= 64) range_step<4>(lo, hi, top);
  if (p.group >= 128) range_step<8>(lo, hi, top);
  constexpr float kMost = static_cast<float>((1 << BITS) - 1);
  float step = round_to<DT>((hi * 0.5f - lo * 0.5f) / kMost * 2.f);
  if (step < 0x1p-100f) step = 0.f;
  const bool finite = top < 0x7f800000u;
  const float inv2 = finite && step > 0.f ? 2.f / step : 0.f;
  const float half = step * 0.5f, quarter = step * 0.25f, lo2 = lo * 0.5f;
  uint32_t word[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float d2 = v[j] * 0.5f - lo2;
    float k = floorf(__builtin_fmaf(d2, inv2, 0.5f));
    const float r = __builtin_fmaf(-k, half, d2);
    k += r >= quarter ? 1.f : 0.f;
    k -= r < -quarter ? 1.f : 0.f;
    k = fminf(fmaxf(k, 0.f), kMost);
    const uint32_t code = inv2 > 0.f ? static_cast<uint32_t>(k) : 0u;
    word[BITS == 4 ? 0 : j >> 2] |= code << (BITS == 4 ? 4 * j : 8 * (j & 3));
  }
  if (!live) return;
  const int64_t to = bh * p.capacity + p.offset + l;
  if constexpr (BITS == 4) {
    s.codes[to * (s.dim >> 3) + c] = word[0];
  } else {
    *reinterpret_cast<uint2*>(s.codes + to * (s.dim >> 2) + 2 * c) = make_uint2(word[0], word[1]);
  }
  if ((c * 8) % p.group == 0) {
    const float nan = __uint_as_float(0x7fc00000u);
    store_pair<DT>(s.params, to * (s.dim / p.group) + c * 8 / p.group, finite ? step : nan, finite ? lo : nan);
  }
}

template <int DT, int KB, int VB>
__global__ __launch_bounds__(256) void affine_append_kernel(const AffineAppendParams p) {
  // dim / 8 is a multiple of group / 8, so a group's lanes are neighbours and a workgroup holds whole groups
  const bool values = blockIdx.x >= p.k_blocks;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) - (values ? p.k_blocks : 0)) * 256 + threadIdx.x;
  if (values) {
    const AffineSide& s = p.side[1];
    append_chunk<DT, VB>(p, s, min(i, s.chunks - 1), i < s.chunks);
  } else {
    const AffineSide& s = p.side[0];
    append_chunk<DT, KB>(p, s, min(i, s.chunks - 1), i < s.chunks);
  }
}

struct AffineBackParams {
  const uint32_t* codes;
  const void* params;
  void* out;
  int64_t chunks;  // B * H * T * dim / 8
  int T, dim, group;
  int64_t capacity;
};

// x = s c + b: s c is exact in f32 for 16-bit s, so the fma rounds once, and the store to the output's type again.
template <int DT, int OT, int BITS>
__global__ __launch_bounds__(256) void affine_dequant_kernel(const AffineBackParams p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.chunks) return;
  const int per_row = p.dim >> 3;
  const int64_t row = i / per_row;
  const int c = static_cast<int>(i - row * per_row);
  const int64_t bh = row / p.T;
  const int64_t at = bh * p.capacity + (row - bh * p.T);
  uint32_t word[2];
  if constexpr (BITS == 4) {
    word[0] = p.codes[at * (p.dim >> 3) + c];
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p.codes + at * (p.dim >> 2) + 2 * c);
    word[0] = u.x, word[1] = u.y;
  }
  const float2 sb = affine_pair<DT>(p.params, at * (p.dim / p.group) + c * 8 / p.group);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t code = BITS == 4 ? (word[0] >> (4 * j)) & 15u : (word[j >> 2] >> (8 * (j & 3))) & 255u;
    v[j] = __builtin_fmaf(sb.x, static_cast<float>(code), sb.y);
  }
  const int64_t to = row * p.dim + c * 8;
  if constexpr (OT == TQ_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + to);
    o[0] = make_float4(v[0], v[1], v[2], v[3]);
    o[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = OT == TQ_DTYPE_F16 ? f32_to_f16_bits(v[2 * j]) | static_cast<uint32_t>(f32_to_f16_bits(v[2 * j + 1])) << 16
                                : f32_to_bf16_bits(v[2 * j]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * j + 1])) << 16;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int DT>
void launch_append(const AffineAppendParams& p, unsigned blocks, hipStream_t st) {
  const int kb = p.side[0].bits, vb = p.side[1].bits;
  if (kb == 4 && vb == 4)
    affine_append_kernel<DT, 4, 4><<<blocks, 256, 0, st>>>(p);
  else if (kb == 8 && vb == 4)
    affine_append_kernel<DT, 8, 4><<<blocks, 256, 0, st>>>(p);
  else if (kb == 4)
    affine_append_kernel<DT, 4, 8><<<blocks, 256, 0, st>>>(p);
  else
    affine_append_kernel<DT, 8, 8><<<blocks, 256, 0, st>>>(p);
}

template <int DT, int OT>
void launch_back(const AffineBackParams& p, int bits, unsigned blocks, hipStream_t st) {
  if (bits == 4)
    affine_dequant_kernel<DT, OT, 4><<<blocks, 256, 0, st>>>(p);
  else
    affine_dequant_kernel<DT, OT, 8><<<blocks, 256, 0, st>>>(p);
}

template <int DT>
void launch_back_to(const AffineBackParams& p, int bits, int out_dtype, unsigned blocks, hipStream_t st) {
  if (out_dtype == TQ_DTYPE_F32)
    launch_back<DT, TQ_DTYPE_F32>(p, bits, blocks, st);
  else if (out_dtype == TQ_DTYPE_F16)
    launch_back<DT, TQ_DTYPE_F16>(p, bits, blocks, st);
  else
    launch_back<DT, TQ_DTYPE_BF16>(p, bits, blocks, st);
}

// TQ_OK, or what is wrong with one side's dim, bits and group.
int check_affine(const char* what, int dim, int bits, int group) {
  if (bits != 4 && bits != 8) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: bits %d are not 4 or 8", what, bits);
  if ((group != 32 && group != 64 && group != 128) || dim < group || dim > 512 || dim % group)
    return fail(TQ_ERR_UNSUPPORTED, "%s: head dim %d in groups of %d (multiples of a group of 32, 64 or 128, to 512)", what, dim, group);
  return TQ_OK;
}

bool aligned16(const void* x, int64_t a, int64_t b, int64_t c, int item) {
  return ((reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>((a | b | c) * item)) & 15) == 0;
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" {

int tq_append_affine_kv(const void* k, const void* v, int dtype, int B, int H, int L, int k_dim, int v_dim,
                        int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_l, int64_t v_stride_b,
                        int64_t v_stride_h, int64_t v_stride_l, int k_bits, int v_bits, int group, uint32_t* k_codes,
                        void* k_params, uint32_t* v_codes, void* v_params, int64_t capacity, int64_t offset,
                        void* stream) {
  const char* what = "tq_append_affine_kv";
  if (dtype < TQ_DTYPE_F32 || dtype > TQ_DTYPE_BF16) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: dtype %d", what, dtype);
  if (B < 0 || H < 0 || L < 0) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: bad sizes B=%d H=%d L=%d", what, B, H, L);
  if (int rc = check_affine(what, k_dim, k_bits, group)) return rc;
  if (int rc = check_affine(what, v_dim, v_bits, group)) return rc;
  if (capacity < 0 || capacity > INT32_MAX || offset < 0 || offset > capacity || L > capacity - offset)
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: tokens %lld + %d over the capacity of %lld", what, static_cast<long long>(offset), L,
                static_cast<long long>(capacity));
  if (B == 0 || H == 0 || L == 0) return TQ_OK;
  if (!k || !v || !k_codes || !k_params || !v_codes || !v_params) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  const int item = dtype == TQ_DTYPE_F32 ? 4 : 2;
  if (!aligned16(k, k_stride_b, k_stride_h, k_stride_l, item) || !aligned16(v, v_stride_b, v_stride_h, v_stride_l, item))
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: vectors and their strides must be 16-byte aligned", what);
  const int64_t rows = static_cast<int64_t>(B) * H * L;
  AffineAppendParams p{};
  p.side[0] = {k, k_stride_b, k_stride_h, k_stride_l, k_codes, k_params, k_dim, k_bits, rows * (k_dim / 8)};
  p.side[1] = {v, v_stride_b, v_stride_h, v_stride_l, v_codes, v_params, v_dim, v_bits, rows * (v_dim / 8)};
  p.k_blocks = (p.side[0].chunks + 255) / 256;
  p.H = H, p.L = L, p.group = group;
  p.capacity = capacity, p.offset = offset;
  const int64_t blocks = p.k_blocks + (p.side[1].chunks + 255) / 256;
  if (blocks > INT32_MAX / 256) return fail(TQ_ERR_UNSUPPORTED, "%s: %lld vectors in one call", what, static_cast<long long>(rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TQ_DTYPE_F32)
    launch_append<TQ_DTYPE_F32>(p, static_cast<unsigned>(blocks), st);
  else if (dtype == TQ_DTYPE_F16)
    launch_append<TQ_DTYPE_F16>(p, static_cast<unsigned>(blocks), st);
  else
    launch_append<TQ_DTYPE_BF16>(p, static_cast<unsigned>(blocks), st);
  return check_launch(what);
}

int tq_dequantize_affine(const uint32_t* codes, const void* params, int dtype, int B, int H, int T, int dim, int bits,
                         int group, int64_t capacity, void* out, int out_dtype, void* stream) {
  const char* what = "tq_dequantize_affine";
  if (dtype < TQ_DTYPE_F32 || dtype > TQ_DTYPE_BF16 || out_dtype < TQ_DTYPE_F32 || out_dtype > TQ_DTYPE_BF16)
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: dtypes %d -> %d", what, dtype, out_dtype);
  if (B < 0 || H < 0 || T < 0 || capacity < T || capacity > INT32_MAX)
    return fail(TQ_ERR_INVALID_ARGUMENT, "%s: bad sizes B=%d H=%d T=%d of %lld", what, B, H, T, static_cast<long long>(capacity));
  if (int rc = check_affine(what, dim, bits, group)) return rc;
  if (B == 0 || H == 0 || T == 0) return TQ_OK;
  if (!codes || !params || !out) return fail(TQ_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  AffineBackParams p{codes, params, out, static_cast<int64_t>(B) * H * T * (dim / 8), T, dim, group, capacity};
  const int64_t blocks = (p.chunks + 255) / 256;
  if (blocks > INT32_MAX / 256)
    return fail(TQ_ERR_UNSUPPORTED, "%s: %lld vectors in one call", what, static_cast<long long>(B) * H * T);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TQ_DTYPE_F32)
    launch_back_to<TQ_DTYPE_F32>(p, bits, out_dtype, static_cast<unsigned>(blocks), st);
  else if (dtype == TQ_DTYPE_F16)
    launch_back_to<TQ_DTYPE_F16>(p, bits, out_dtype, static_cast<unsigned>(blocks), st);
  else
    launch_back_to<TQ_DTYPE_BF16>(p, bits, out_dtype, static_cast<unsigned>(blocks), st);
  return check_launch(what);
}

}  // extern "C"
