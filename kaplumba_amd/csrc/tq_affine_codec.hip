// The group-affine cache's write and read back.
#include <algorithm>

#include "tq_affine.h"

namespace tq {
namespace {

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 by one multiplication: m = ceil(2^(31 + k) / d), 2^k >= d, is under 2^32
// and n m / 2^(31 + k) exceeds n / d by less than 1 / d.
struct Divisor {
  uint32_t d, m, shift;
};

Divisor divisor(int64_t d) {
  uint32_t k = 0;
  while ((int64_t{1} << k) < d) ++k;
  return {static_cast<uint32_t>(d), static_cast<uint32_t>(((uint64_t{1} << (31 + k)) + d - 1) / d), 31 + k};
}

__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor& d) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * d.m) >> d.shift);
}

// One side (keys or values) of an append.
struct AffineSide {
  const void* x;
  int64_t sb, sh, sl;
  uint32_t* codes;
  void* params;
  int dim, bits;
  Divisor per_row;   // pieces of 16 coordinates a row
  uint32_t chunks;   // of all rows, under 2^31
};

struct AffineAppendParams {
  AffineSide side[2];
  uint32_t k_blocks;  // workgroups of the keys; the rest are the values'
  Divisor H, L;
  int group;
  int64_t capacity, offset;
};

// Eight consecutive elements of x as f32, in 16-byte loads where the host found them aligned.
template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t at, float* v) {
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
__device__ __forceinline__ void range_step(float& lo, float& hi, float& odd) {
  lo = fminf(lo, xor_lane<OFF>(lo));
  hi = fmaxf(hi, xor_lane<OFF>(hi));
  odd += xor_lane<OFF>(odd);
}

// A lane holds 16 coordinates of one row, two pieces of eight half a group apart (so that neighbouring lanes load and
// store neighbouring bytes), group / 16 neighbouring lanes a group:
//   lo, hi = the group's least and greatest value, s = T((hi - lo) / n), n = 2^bits - 1, bias = lo,
//   code = the number of half steps (k + 1/2) s, k = 0 .. n - 1, that d = x - lo (in f32) reaches.
// Differences are taken in halves, so that they stay finite.  d / s lies within an ulp of d * (1 / s); the residual
// d - k s is exact in an fma (both are multiples of ulp(s) and it is at most s), which settles the border, so the
// hardware's reciprocal (off by an ulp) is enough.
// Scales below 2^-100 count as 0 (every code 0), so that 1 / s and the halves stay normal.
// s and bias are of the vectors' own type: lo is then exact, and s off by half a step at most over the whole
// range (2^-9 of it in bf16, 1/255 of it is a step at 8 bits).  A group with a value that is not finite gets NaN
// for both, and codes of 0.
// Bound by memory, and by a launch's first round of loads: 8192 tokens of 2 x 8 heads of 128, bf16 at 4 bits (43 MB),
// 12.6 us, 3.4 TB/s; eight coordinates a lane and divisions by hand were 22 us.
template <int DT, int BITS>
__device__ __forceinline__ void append_chunk(const AffineAppendParams& p, const AffineSide& s, uint32_t i, bool live) {
  const uint32_t row = quotient(i, s.per_row);
  const int c = static_cast<int>(i - row * s.per_row.d);
  const uint32_t bh = quotient(row, p.L);
  const uint32_t l = row - bh * p.L.d;
  const uint32_t b = quotient(bh, p.H);
  const uint32_t h = bh - b * p.H.d;
  float v[16];
  const int shift = p.group == 32 ? 1 : p.group == 64 ? 2 : 3;  // lanes a group
  const int in_group = c & ((1 << shift) - 1), g = c >> shift;
  const int at = g * p.group + in_group * 8;
  const int64_t from = b * s.sb + h * s.sh + l * s.sl + at;
  load8<DT>(s.x, from, v);
  load8<DT>(s.x, from + (p.group >> 1), v + 8);
  float lo = v[0], hi = v[0], odd = 0.f;  // odd: 0 times every value, NaN where one is not finite
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    lo = fminf(lo, v[j]);
    hi = fmaxf(hi, v[j]);
    odd = __builtin_fmaf(v[j], 0.f, odd);
  }
  range_step<1>(lo, hi, odd);
  if (p.group >= 64) range_step<2>(lo, hi, odd);
  if (p.group >= 128) range_step<4>(lo, hi, odd);
  constexpr float kMost = static_cast<float>((1 << BITS) - 1);
  float step = round_to<DT>((hi * 0.5f - lo * 0.5f) / kMost * 2.f);
  if (step < 0x1p-100f) step = 0.f;
  const bool finite = odd == 0.f;
  const bool codes = finite && step > 0.f;
  const float inv2 = codes ? 2.f * __builtin_amdgcn_rcpf(step) : 0.f;
  const float half = step * 0.5f, quarter = codes ? step * 0.25f : INFINITY, lo2 = lo * 0.5f;
  uint32_t word[BITS / 2] = {};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float d2 = __builtin_fmaf(v[j], 0.5f, -lo2);
    const float k = floorf(__builtin_fmaf(d2, inv2, 0.5f));
    const float r = __builtin_fmaf(-k, half, d2);
    int code = static_cast<int>(fminf(fmaxf(k, 0.f), kMost));  // in range for NaN too
    code += r >= quarter ? 1 : 0;
    code -= r < -quarter ? 1 : 0;
    word[j * BITS / 32] |= static_cast<uint32_t>(min(code, (1 << BITS) - 1)) << (j * BITS % 32);
  }
  if (!live) return;
  const int64_t to = bh * p.capacity + p.offset + l;
  uint32_t* piece = s.codes + to * (s.dim * BITS / 32) + at * BITS / 32;
  if constexpr (BITS == 4) {
    piece[0] = word[0];
    piece[p.group >> 4] = word[1];
  } else {
    *reinterpret_cast<uint2*>(piece) = make_uint2(word[0], word[1]);
    *reinterpret_cast<uint2*>(piece + (p.group >> 3)) = make_uint2(word[2], word[3]);
  }
  if (in_group == 0) {
    const float nan = __uint_as_float(0x7fc00000u);
    store_pair<DT>(s.params, to * (s.dim >> (shift + 4)) + g, finite ? step : nan, finite ? lo : nan);
  }
}

template <int DT, int KB, int VB>
__global__ __launch_bounds__(256) void affine_append_kernel(const AffineAppendParams p) {
  // dim / 16 is a multiple of group / 16, so a group's lanes are neighbours and a workgroup holds whole groups
  const bool values = blockIdx.x >= p.k_blocks;
  const uint32_t i = (blockIdx.x - (values ? p.k_blocks : 0)) * 256 + threadIdx.x;
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
  uint32_t chunks;  // pieces of eight coordinates: B * H * T * dim / 8, under 2^31
  Divisor per_row, T;
  int dim, group;
  int64_t capacity;
};

// x = s c + b: s c is exact in f32 for 16-bit s, so the fma rounds once, and the store to the output's type again.
// Bound by memory: a side of 8192 tokens of 8 heads of 128, 4 bits to bf16 (21 MB), 6.3 us, 3.4 TB/s with the launch.
template <int DT, int OT, int BITS>
__global__ __launch_bounds__(256) void affine_dequant_kernel(const AffineBackParams p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.chunks) return;
  const uint32_t row = quotient(i, p.per_row);
  const int c = static_cast<int>(i - row * p.per_row.d);
  const uint32_t bh = quotient(row, p.T);
  const int64_t at = bh * p.capacity + (row - bh * p.T.d);
  const int shift = p.group == 32 ? 2 : p.group == 64 ? 3 : 4;  // pieces a group
  uint32_t word[2];
  if constexpr (BITS == 4) {
    word[0] = p.codes[at * (p.dim >> 3) + c];
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p.codes + at * (p.dim >> 2) + 2 * c);
    word[0] = u.x, word[1] = u.y;
  }
  const float2 sb = affine_pair<DT>(p.params, at * (p.dim >> (shift + 3)) + (c >> shift));
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t code = (word[j * BITS / 32] >> (j * BITS % 32)) & ((1u << BITS) - 1u);
    v[j] = __builtin_fmaf(sb.x, static_cast<float>(code), sb.y);
  }
  const int64_t to = static_cast<int64_t>(row) * p.dim + c * 8;
  if constexpr (OT == TQ_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + to);
    o[0] = make_float4(v[0], v[1], v[2], v[3]);
    o[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (OT == TQ_DTYPE_F16) {
        typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
        const half2_t t = {static_cast<_Float16>(v[2 * j]), static_cast<_Float16>(v[2 * j + 1])};
        w[j] = __builtin_bit_cast(uint32_t, t);
      } else {
        typedef __bf16 bhalf2_t __attribute__((ext_vector_type(2)));
        const bhalf2_t t = {static_cast<__bf16>(v[2 * j]), static_cast<__bf16>(v[2 * j + 1])};
        w[j] = __builtin_bit_cast(uint32_t, t);
      }
    }
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
  if (rows > INT32_MAX / (std::max(k_dim, v_dim) / 16))
    return fail(TQ_ERR_UNSUPPORTED, "%s: %lld vectors in one call", what, static_cast<long long>(rows));
  AffineAppendParams p{};
  p.side[0] = {k, k_stride_b, k_stride_h, k_stride_l, k_codes, k_params, k_dim, k_bits, divisor(k_dim / 16),
               static_cast<uint32_t>(rows * (k_dim / 16))};
  p.side[1] = {v, v_stride_b, v_stride_h, v_stride_l, v_codes, v_params, v_dim, v_bits, divisor(v_dim / 16),
               static_cast<uint32_t>(rows * (v_dim / 16))};
  p.k_blocks = (p.side[0].chunks + 255) / 256;
  p.H = divisor(H), p.L = divisor(L), p.group = group;
  p.capacity = capacity, p.offset = offset;
  const uint32_t blocks = p.k_blocks + (p.side[1].chunks + 255) / 256;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TQ_DTYPE_F32)
    launch_append<TQ_DTYPE_F32>(p, blocks, st);
  else if (dtype == TQ_DTYPE_F16)
    launch_append<TQ_DTYPE_F16>(p, blocks, st);
  else
    launch_append<TQ_DTYPE_BF16>(p, blocks, st);
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
  const int64_t rows = static_cast<int64_t>(B) * H * T;
  if (rows > INT32_MAX / (dim / 8))
    return fail(TQ_ERR_UNSUPPORTED, "%s: %lld vectors in one call", what, static_cast<long long>(rows));
  AffineBackParams p{codes, params, out, static_cast<uint32_t>(rows * (dim / 8)), divisor(dim / 8), divisor(T), dim, group,
                     capacity};
  const uint32_t blocks = (p.chunks + 255) / 256;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TQ_DTYPE_F32)
    launch_back_to<TQ_DTYPE_F32>(p, bits, out_dtype, blocks, st);
  else if (dtype == TQ_DTYPE_F16)
    launch_back_to<TQ_DTYPE_F16>(p, bits, out_dtype, blocks, st);
  else
    launch_back_to<TQ_DTYPE_BF16>(p, bits, out_dtype, blocks, st);
  return check_launch(what);
}

}  // extern "C"
